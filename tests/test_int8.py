"""8-bit integer linears: quantiser, products, gated block and their gradients, against a plain
implementation in 64 bits.

Tolerances.  A rounding to a type t is off by at most eps_t / 2 of the value.  The epilogues
take a handful of fp32 steps (2^-24 each) before the one rounding to the output type; the
gradients' digits are off by at most half a step of the row maximum / V_P, summed over the
contraction.  Every bound below is formed element by element from these, in 64 bits.
"""

from __future__ import annotations

import copy
import math

import pytest
import torch

from int_model_approximation_b200 import _native as nat
from int_model_approximation_b200 import int8, students, synthetic
from int_model_approximation_b200.freivalds import freivalds_vector, verify_int32_product

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ACTS = ["silu", "gelu", "gelu_tanh"]
U32 = 2.0**-24


# ---------------------------------------------------------------------------
# plain forms, 64 bits
# ---------------------------------------------------------------------------
def plain_codes(x):
    """(codes, scale) as float64: both quotients rounded to fp32, as the definition says."""
    x = x.detach().double()
    amax = x.abs().amax(dim=1) if x.shape[1] else torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
    s = (amax / 127.0).float().clamp_min(1e-12).double()
    q = (x / s[:, None]).float().round().clamp(-127, 127).double()
    return q, s


def plain_act(g, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g**3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 0.134145 * g * g)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the distance of the subnormals: what a rounding near zero may be off."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def digit_limit(*dtypes):
    return 32639.0 if all(t == torch.bfloat16 for t in dtypes) else 8355711.0


def assert_within(got, want, bound):
    d = (got.double() - want).abs()
    bad = ~(d <= bound)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} outside; first at {i}: got {got[i].item()}, want "
                             f"{want[i].item()}, bound {bound[i].item()}")


def make(m, n, k, dtype, seed, dev, bias=False):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = synthetic.student_t_activations(m, k, seed, device=dev).to(dtype)
    w = (torch.randn((n, k), generator=g, device=dev) * 0.05).to(dtype)
    b = (torch.randn((n,), generator=g, device=dev) * 0.1).to(dtype) if bias else None
    return x, w, b


def pre(q, s, w, t, b):
    """The rescaled product and the sum of the magnitudes it was added from."""
    y = (q @ w.T) * s[:, None] * t
    mag = y.abs()
    if b is not None:
        y, mag = y + b.double(), mag + b.double().abs()
    return y, mag


def status_clean(dev):
    assert nat.device_status(dev.index or 0, clear=True) == (0, 0, 0)


# ---------------------------------------------------------------------------
# refusals (no launch, no GPU)
# ---------------------------------------------------------------------------
def test_host_tensors_are_refused():
    x, w = torch.zeros(2, 16), torch.zeros(4, 16)
    with pytest.raises(RuntimeError, match="no CPU execution path"):
        int8.per_token_int8(x)
    with pytest.raises(RuntimeError, match="no CPU execution path"):
        int8.int8_linear(x, w)
    with pytest.raises(RuntimeError, match="no CPU execution path"):
        int8.int8_gated(x, w, w)
    with pytest.raises(RuntimeError, match="no CPU execution path"):
        int8.int8_gemm(x.to(torch.int8), w.to(torch.int8))
    with pytest.raises(RuntimeError, match="no CPU execution path"):
        int8.Int8Weight(w.to(torch.int8), torch.ones(4))
    with pytest.raises(RuntimeError, match="no CPU execution path"):
        int8.Int8Weight.from_float(w)
    with pytest.raises(RuntimeError, match="no CPU execution path"):
        students.Int8Linear(w, None)


def test_float_operands_of_the_int8_product_are_refused():
    with pytest.raises(RuntimeError, match="2-D int8"):
        int8.int8_gemm(torch.zeros(2, 16), torch.zeros(4, 16, dtype=torch.int8))
    with pytest.raises(RuntimeError, match="2-D int8"):
        int8.int8_gemm(torch.zeros(2, 2, 16, dtype=torch.int8), torch.zeros(4, 16, dtype=torch.int8))


def test_c_entries_refuse_bad_arguments_before_any_launch():
    lib = nat.lib()
    bad = nat.IMA_ERR_INVALID_ARGUMENT
    uns = nat.IMA_ERR_UNSUPPORTED
    # row stride below K, not a multiple of 16, pointer not on 16 bytes, unknown type, no scale
    assert lib.ima_int8_quantize_rows(16, 1, 2, 32, 32, 16, 16, 16, None) == bad
    assert lib.ima_int8_quantize_rows(16, 1, 2, 20, 20, 16, 24, 16, None) == bad
    assert lib.ima_int8_quantize_rows(16, 1, 2, 32, 32, 17, 32, 16, None) == bad
    assert lib.ima_int8_quantize_rows(16, 9, 2, 32, 32, 16, 32, 16, None) == bad
    assert lib.ima_int8_quantize_rows(16, 1, 2, 32, 32, 16, 32, None, None) == bad
    # product: no output, y without scales, contraction too long, misaligned operand
    assert lib.ima_int8_gemm(16, 32, 16, 32, 2, 2, 32, None, 2, None, None, None, 0, None, 0, 2, None) == bad
    assert lib.ima_int8_gemm(16, 32, 16, 32, 2, 2, 32, None, 2, None, None, None, 0, 16, 1, 2, None) == bad
    assert lib.ima_int8_gemm(16, 131072, 16, 131072, 2, 2, 131072, 16, 2, None, None, None, 0, None, 0, 2, None) == uns
    assert lib.ima_int8_gemm(24, 32, 16, 32, 2, 2, 32, 16, 2, None, None, None, 0, None, 0, 2, None) == bad
    assert lib.ima_int8_gemm(16, 24, 16, 32, 2, 2, 24, 16, 2, None, None, None, 0, None, 0, 2, None) == bad
    assert lib.ima_int8_gemm(16, 32, 16, 32, 2, 2, 32, 16, 1, None, None, None, 0, None, 0, 2, None) == bad
    # gated: unknown activation
    assert lib.ima_int8_gated(16, 1, 2, 32, 32, 16, 32, 16, 0, 16, 32, 16, 32, 2, 16, 16, None, 0, None, 0, 0, None, None, 0,
                              7, 16, 2, None) == uns
    # backward: only 2 or 3 digits, contractions too long, no workspace
    def backward(m=2, n=32, k=32, planes=2, dx=256, dw=None, ws=256):
        ld = (max(n, k) + 15) // 16 * 16
        return lib.ima_int8_linear_backward(16, 1, n, m, n, k, 16, ld, 16, 16, ld, 16, ld, 16, planes, dx, 1, dw, 1, None,
                                            1, ws, None)
    assert backward(planes=1) == uns and backward(n=131072) == uns and backward(m=131072, dx=None, dw=256) == uns
    assert backward(ws=None) == bad


@pytest.mark.gpu
def test_mismatched_calls_are_refused(cuda_device):
    x, w, b = make(4, 8, 32, torch.bfloat16, 0, cuda_device, bias=True)
    w2 = int8.Int8Weight.from_float(w[:, :16])
    with pytest.raises(RuntimeError, match="shape mismatch"):
        int8.int8_linear(x, w2)
    with pytest.raises(RuntimeError, match="shape mismatch"):
        int8.int8_gated(x, w2, w2)
    with pytest.raises(RuntimeError, match="differ in shape"):
        int8.int8_gated(x, w, w[:4])
    with pytest.raises(RuntimeError, match="unknown activation"):
        int8.int8_gated(x, w, w, activation="relu6")
    with pytest.raises(RuntimeError, match="entries, expected"):
        int8.int8_linear(x, w, b[:3])
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        int8.int8_linear(x, w, b.cpu())
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        int8.int8_linear(x.double(), w)
    q = torch.zeros((4, 32), dtype=torch.int8, device=cuda_device)
    with pytest.raises(RuntimeError, match="needs x_scale and w_scale"):
        int8.int8_gemm(q, q, y_dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no output"):
        int8.int8_gemm(q, q, want_c=False)
    with pytest.raises(RuntimeError, match="int8 product"):
        int8.int8_gemm(q, q, c_out=torch.empty((4, 4), dtype=torch.int64, device=cuda_device))
    with pytest.raises(RuntimeError, match="contiguous rows"):
        int8.int8_gemm(q, q, c_out=torch.empty((4, 4), dtype=torch.int32, device=cuda_device).t())
    long = torch.zeros((1, int8.MAX_K + 1), dtype=torch.int8, device=cuda_device)
    with pytest.raises(RuntimeError, match="exceeds"):
        int8.int8_gemm(long, long)
    status_clean(cuda_device)


# ---------------------------------------------------------------------------
# quantiser
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (9, 16), (33, 1000), (5, 1024), (4, 1025), (7, 4096), (3, 4099),
                                 (2, 20480), (3, 20491), (600, 64)])
def test_quantiser_matches_its_definition(cuda_device, dtype, m, k):
    x = synthetic.student_t_activations(m, k, 17 + m + k, device=cuda_device, outlier_fraction=0.01).to(dtype)
    q, s = int8.per_token_int8(x)
    q64, s64 = plain_codes(x)
    assert torch.equal(s.flatten().double(), s64)
    assert torch.equal(q.double(), q64)
    # a view whose rows are not 16-byte aligned
    wide = torch.zeros((m, k + 3), dtype=dtype, device=cuda_device)
    wide[:, 1:k + 1] = x
    q2, s2 = int8.per_token_int8(wide[:, 1:k + 1])
    assert torch.equal(q2, q) and torch.equal(s2, s)
    status_clean(cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 7), (torch.float16, 10)])
@pytest.mark.parametrize("k_pad", [0, 5])
def test_quantiser_every_pair_of_significands(cuda_device, dtype, bits, k_pad):
    """Codes against torch's fp32 division for every significand of the row maximum and of the
    element, over the ten binades in which the code is not 0 whatever the rounding.  Other rows
    differ by powers of two, which scale every step exactly.  k_pad 5: rows off the 16-byte grid."""
    n = 2**bits
    maxima = (1.0 + torch.arange(n, device=cuda_device) / n) * 2.0
    binades = 2.0 ** torch.arange(1, -9, -1, device=cuda_device).float()
    elements = ((1.0 + torch.arange(n, device=cuda_device) / n)[None] * binades[:, None]).reshape(-1)
    for chunk in maxima.split(128):
        x = torch.zeros((chunk.numel(), elements.numel() + 1 + k_pad), device=cuda_device, dtype=dtype)
        x[:, 0] = chunk.to(dtype)
        rest = elements[None].expand(chunk.numel(), -1) * (elements[None] <= chunk[:, None])
        sign = torch.where(torch.arange(elements.numel(), device=cuda_device) % 3 == 0, -1.0, 1.0)
        x[:, 1:1 + elements.numel()] = (rest * sign).to(dtype)
        q, s = int8.per_token_int8(x)
        x32 = x.float()
        s32 = x32.abs().amax(dim=1, keepdim=True) / torch.full_like(s, 127.0)
        assert torch.equal(s, s32)
        assert torch.equal(q.float(), (x32 / s32).round())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantiser_ties_and_special_rows(cuda_device, dtype):
    rows = torch.zeros((9, 40), dtype=torch.float32)
    rows[0, :32] = torch.arange(32) + 0.5        # with amax 127: scale 1, every element a tie
    rows[0, 33] = 127.0
    rows[1, :32] = -(torch.arange(32) + 0.5)
    rows[1, 33] = -127.0
    rows[2] = 0.0                                # scale 1e-12, codes 0
    rows[3, 5] = 1e-14                           # below the smallest scale
    rows[4, 7] = float("nan")
    rows[4, 8] = 3.0
    rows[5, 1] = float("inf")
    rows[5, 2] = 2.0
    rows[6, 1] = float("-inf")
    rows[7, :] = torch.finfo(dtype).max
    rows[8, 0], rows[8, 1] = 1.0, -1.0
    x = rows.to(dtype).to(cuda_device)
    q, s = int8.per_token_int8(x)
    keep = [0, 1, 2, 3, 7, 8]
    q64, s64 = plain_codes(x[keep])
    assert torch.equal(q[keep].double(), q64) and torch.equal(s[keep].flatten().double(), s64)
    assert torch.isnan(s[4]) and torch.isinf(s[5]) and torch.isinf(s[6])
    assert int(q[4:7].abs().max()) == 0
    # such rows come out as NaN and leave the others alone
    w = int8.Int8Weight.from_float(torch.randn((24, 40), device=cuda_device))
    y = int8.int8_linear(x, w)
    assert torch.isnan(y[4:7]).all() and torch.isfinite(y[:4].float()).all()
    status_clean(cuda_device)


# ---------------------------------------------------------------------------
# the integer product
# ---------------------------------------------------------------------------
def int_product(a, b):
    """The exact product: float64 is exact to 2^53."""
    return (a.double() @ b.double().T).to(torch.int32)


# One token to several tiles per CTA; the last ones reach single CTAs, then CTA pairs with several tiles
# each, those before the split form with few and many tokens.
SHAPES = [(1, 1, 1), (8, 18944, 128), (100, 130, 2500), (128, 64, 20000), (513, 300, 5000), (1, 4864, 896), (2, 130, 4099), (5, 3, 17), (16, 896, 4864), (17, 64, 128), (33, 1009, 257),
          (64, 129, 1000), (65, 256, 128), (127, 255, 129), (128, 256, 512), (129, 257, 640), (257, 513, 896),
          (300, 128, 4864), (1000, 200, 72),
          (300, 10250, 136), (3000, 4001, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_int8_product_is_exact(cuda_device, m, n, k):
    g = torch.Generator(device=cuda_device).manual_seed(m + n + k)
    a = torch.randint(-128, 128, (m, k), generator=g, device=cuda_device, dtype=torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=g, device=cuda_device, dtype=torch.int8)
    c, y = int8.int8_gemm(a, b)
    assert y is None and torch.equal(c, int_product(a, b))
    status_clean(cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 300])
def test_int8_product_longest_contraction_of_extremes(cuda_device, m):
    k = int8.MAX_K
    a = torch.full((m, k), -128, dtype=torch.int8, device=cuda_device)
    b = torch.full((3, k), -128, dtype=torch.int8, device=cuda_device)
    b[1] = 127
    c, _ = int8.int8_gemm(a, b)
    want = torch.tensor([128 * 128 * k, -128 * 127 * k, 128 * 128 * k], device=cuda_device)
    assert torch.equal(c.long(), want.expand(m, 3))
    status_clean(cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 30, 150])
def test_int8_product_strides_outputs_and_neighbours(cuda_device, m):
    """Transposed and sliced operands; outputs inside larger tensors, whose other elements stay."""
    n, k = 77, 200
    g = torch.Generator(device=cuda_device).manual_seed(5)
    big = torch.randint(-128, 128, (k + 5, m + 9), generator=g, device=cuda_device, dtype=torch.int8)
    a = big[2:k + 2, 3:m + 3].t()
    b = torch.randint(-128, 128, (n, 2 * k), generator=g, device=cuda_device, dtype=torch.int8)[:, ::2]
    want = int_product(a, b)
    xs = torch.rand((m, 1), generator=g, device=cuda_device) + 0.5
    ws = torch.rand((n,), generator=g, device=cuda_device) + 0.5
    c_big = torch.full((m + 4, n + 6), 7, dtype=torch.int32, device=cuda_device)
    y_big = torch.full((m + 4, n + 5), 7.0, dtype=torch.bfloat16, device=cuda_device)
    c, y = int8.int8_gemm(a, b, x_scale=xs, w_scale=ws, c_out=c_big[1:m + 1, 3:n + 3], y_out=y_big[1:m + 1, 1:n + 1])
    assert torch.equal(c, want)
    ref = want.double() * xs.double() * ws.double()
    assert_within(y, ref, (half_step(torch.bfloat16) + 4 * U32) * ref.abs())
    c_big[1:m + 1, 3:n + 3] = 7
    y_big[1:m + 1, 1:n + 1] = 7.0
    assert bool((c_big == 7).all()) and bool((y_big == 7.0).all())
    status_clean(cuda_device)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cuda_device):
    """Outputs and activations of more than 2^31 elements, compared on rows at both ends."""
    m, n, k = 66_000, 33_000, 48
    g = torch.Generator(device=cuda_device).manual_seed(2)
    a = torch.randint(-127, 128, (m, k), generator=g, device=cuda_device, dtype=torch.int8)
    b = torch.randint(-127, 128, (n, k), generator=g, device=cuda_device, dtype=torch.int8)
    ones_m, ones_n = torch.ones((m,), device=cuda_device), torch.ones((n,), device=cuda_device)
    _c, y = int8.int8_gemm(a, b, want_c=False, x_scale=ones_m, w_scale=ones_n, y_dtype=torch.float16)
    pick = torch.tensor([0, 1, 32_999, 65_076, 65_077, m - 2, m - 1], device=cuda_device)
    # 127^2 * 48 exceeds fp16's range: the same rounding, to infinity too
    assert torch.equal(y[pick], int_product(a[pick], b).to(torch.float16))
    q, s = int8.per_token_int8(y.nan_to_num_(posinf=60000.0, neginf=-60000.0))
    q64, s64 = plain_codes(y[pick])
    assert torch.equal(q[pick].double(), q64) and torch.equal(s[pick].flatten().double(), s64)
    del y
    status_clean(cuda_device)


@pytest.mark.gpu
def test_results_under_an_sm_limit(cuda_device):
    """Fewer SMs (left to collectives) give the same results, whatever form or split that selects."""
    x, w, _ = make(700, 3000, 2100, torch.bfloat16, 41, cuda_device)
    x.requires_grad_()
    wt = int8.Int8Weight.from_float(w)
    dy = torch.randn((700, 3000), device=cuda_device).to(torch.bfloat16)

    def run():
        y = int8.int8_linear(x, wt)
        return y, torch.autograd.grad(y, x, dy)[0], int8.int8_linear(x.detach()[:5], wt)

    want = run()
    try:
        for limit in (1, 7, 100):
            nat.call("ima_set_gemm_sm_limit", limit)
            assert all(torch.equal(a, b) for a, b in zip(run(), want))
    finally:
        nat.call("ima_set_gemm_sm_limit", 0)
    status_clean(cuda_device)


@pytest.mark.gpu
def test_int8_product_verifies_under_freivalds(cuda_device):
    x, w, _ = make(50, 96, 300, torch.bfloat16, 3, cuda_device)
    (q, _s), wt = int8.per_token_int8(x), int8.Int8Weight.from_float(w)
    c, _ = int8.int8_gemm(q, wt.codes)
    r = freivalds_vector(96, 4, cuda_device)
    args = q.to(torch.int32).contiguous(), wt.codes.to(torch.int32).t().contiguous()
    assert verify_int32_product(*args, c.long(), r)
    c[17, 3] += 1
    assert not verify_int32_product(*args, c.long(), r)


# ---------------------------------------------------------------------------
# linear and gated, forward
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("bias", [False, True])
def test_linear_forward(cuda_device, dtype, m, n, k, bias):
    x, w, b = make(m, n, k, dtype, m * 7 + n, cuda_device, bias)
    (q, s), (wq, t) = plain_codes(x), plain_codes(w)
    want, mag = pre(q, s, wq, t, b)
    bound = half_step(dtype) * want.abs() + 6 * U32 * mag + smallest(dtype)
    y = int8.int8_linear(x, int8.Int8Weight.from_float(w), b)
    assert y.dtype == dtype
    assert_within(y, want, bound)
    assert torch.equal(int8.int8_linear(x, w, b), y)           # the same weight quantised in the call
    status_clean(cuda_device)


def gated_reference(x, w1, w2, b1, b2, act):
    q, s = plain_codes(x)
    (q1, t1), (q2, t2) = plain_codes(w1), plain_codes(w2)
    g, gm = pre(q, s, q1, t1, b1)
    u, um = pre(q, s, q2, t2, b2)
    a, da = plain_act(g, act)
    return dict(q=q, s=s, q1=q1, t1=t1, q2=q2, t2=t2, g=g, gm=gm, u=u, um=um, a=a, da=da)


# The activation and its derivative in fp32.  exp carries 2 + |1.16 g| units in the last place (its
# documented bound), erfc, tanh and the divisions a few: for |g| <= 40 at most 64 units of 2^-23 on
# a value whose own size is at most |g| + 1.  Beyond |g| = 40 the activations are g or 0 and their
# derivatives 1 or 0 to within 40 e^-40 < 2^-50, whatever the exponential's error.  The derivatives
# of the activations are at most 1.13 and their second derivatives at most 1, which carries the
# error of g itself.
def act_slack(ref, factor=1.0):
    return factor * 64 * 2.0**-23 * (ref["g"].abs() + 1) + 6 * U32 * 1.13 * ref["gm"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, "silu"), (torch.bfloat16, "gelu"), (torch.float16, "gelu_tanh"),
                                       (torch.float32, "silu"), (torch.float32, "gelu"), (torch.float32, "gelu_tanh")])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 4864, 896), (2, 65, 33), (16, 130, 640), (45, 1000, 129), (64, 64, 256),
                                   (65, 127, 896), (130, 129, 300), (300, 896, 128), (300, 5130, 136),
                                   (3000, 2001, 256)])
def test_gated_forward(cuda_device, dtype, act, m, n, k):
    x, w1, b1 = make(m, n, k, dtype, m + n, cuda_device, bias=m % 2 == 0)
    _x, w2, b2 = make(m, n, k, dtype, m + n + 1, cuda_device, bias=m % 2 == 0)
    ref = gated_reference(x, w1, w2, b1, b2, act)
    want = ref["a"] * ref["u"]
    bound = half_step(dtype) * want.abs() + act_slack(ref) * ref["u"].abs() + 8 * U32 * ref["a"].abs() * ref["um"] + \
        2 * U32 * want.abs() + smallest(dtype)
    h = int8.int8_gated(x, int8.Int8Weight.from_float(w1), int8.Int8Weight.from_float(w2), b1, b2, activation=act)
    assert h.dtype == dtype
    assert_within(h, want, bound)
    status_clean(cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 200])
def test_gated_saturated_activations(cuda_device, m):
    """Large |g| on both sides: exp overflows to infinity or vanishes, h must not become NaN."""
    x = torch.ones((m, 64), device=cuda_device)
    w = torch.zeros((8, 64), device=cuda_device)
    w[0], w[1], w[2] = 10.0, -10.0, 1000.0
    w[3] = -1000.0
    up = torch.ones((8, 64), device=cuda_device)
    for act in ACTS:
        h = int8.int8_gated(x, w, up, activation=act)
        assert torch.isfinite(h).all()
        assert torch.allclose(h[:, 0], torch.full((m,), 640.0 * 64, device=cuda_device), rtol=1e-5)
        assert float(h[:, 1].abs().max()) == 0.0 and float(h[:, 3].abs().max()) == 0.0


@pytest.mark.gpu
def test_empty_sizes(cuda_device):
    dev = cuda_device
    for m, n, k in [(0, 5, 32), (3, 0, 32), (3, 5, 0), (0, 0, 0), (200, 5, 0)]:
        x = torch.randn((m, k), device=dev, requires_grad=True)
        w = torch.randn((n, k), device=dev, requires_grad=True)
        w2 = torch.randn((n, k), device=dev, requires_grad=True)
        b = torch.randn((n,), device=dev, requires_grad=True)
        y = int8.int8_linear(x, w, b)
        assert y.shape == (m, n)
        if k == 0:
            assert torch.equal(y, b.expand(m, n))
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
        assert gx.shape == x.shape and gw.shape == w.shape
        assert float(gw.abs().sum()) == 0.0 if m == 0 else torch.isfinite(gw).all()
        assert torch.equal(gb, torch.full((n,), float(m), device=dev))
        if n == 0:
            assert float(gx.abs().sum()) == 0.0
        h = int8.int8_gated(x, w, w2, b, None)
        assert h.shape == (m, n)
        if k == 0:
            assert float(h.detach().abs().sum()) == 0.0
        grads = torch.autograd.grad(h, (x, w, w2, b), torch.ones_like(h))
        assert [g.shape for g in grads] == [x.shape, w.shape, w2.shape, b.shape]
        assert all(bool(torch.isfinite(g).all()) for g in grads)
    status_clean(dev)


# ---------------------------------------------------------------------------
# gradients against the formula
# ---------------------------------------------------------------------------
def grad_bound(d, d_err, factor, codes, limit, dtype, want):
    """Bound of sum_j (d_ij factor_j) codes_jk computed from digits of d against its row maximum.

    d_err: bound on d's own error.  Half a digit step of the row maximum per summand (1.001: the
    rounding of the scale and of the quotient), d's error, fp32 products, the final rounding."""
    v = d * factor
    step = 0.5 * 1.001 * (v.abs().amax(dim=1, keepdim=True) if v.shape[1] else 0) / limit
    size = v.abs() @ codes.abs()
    return step * codes.abs().sum(dim=0) + (d_err * factor.abs()) @ codes.abs() + 6 * U32 * size + \
        half_step(dtype) * want.abs() + smallest(dtype)


GRAD_SHAPES = [(1, 1, 1), (1, 300, 64), (5, 17, 33), (64, 130, 250), (130, 257, 129), (300, 64, 896), (257, 896, 128),
               (300, 64, 10250), (2000, 96, 4000), (2000, 2100, 2500)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", GRAD_SHAPES)
@pytest.mark.parametrize("frozen", [False, True])
def test_linear_gradients(cuda_device, dtype, m, n, k, frozen):
    x, w, b = make(m, n, k, dtype, m + 3 * n, cuda_device, bias=True)
    g = torch.Generator(device=cuda_device).manual_seed(9)
    dy = (torch.randn((m, n), generator=g, device=cuda_device) *
          torch.exp(torch.randn((m, 1), generator=g, device=cuda_device))).to(dtype)
    x.requires_grad_()
    b.requires_grad_()
    (q, s), (wq, t) = plain_codes(x), plain_codes(w)
    if frozen:
        y = int8.int8_linear(x, int8.Int8Weight.from_float(w), b)
        dx, db = torch.autograd.grad(y, (x, b), dy)
    else:
        w.requires_grad_()
        y = int8.int8_linear(x, w, b)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        want = (dy.double() * s[:, None]).T @ q
        none = torch.zeros((n, m), dtype=torch.float64, device=cuda_device)
        assert dw.dtype == dtype
        assert_within(dw, want, grad_bound(dy.double().T, none, s, q, digit_limit(dtype), dtype, want))
    want = (dy.double() * t) @ wq
    none = torch.zeros((m, n), dtype=torch.float64, device=cuda_device)
    assert dx.dtype == dtype and db.dtype == dtype
    assert_within(dx, want, grad_bound(dy.double(), none, t, wq, digit_limit(dtype), dtype, want))
    want = dy.double().sum(dim=0)
    assert_within(db, want, half_step(dtype) * want.abs() + (m + 2) * U32 * dy.double().abs().sum(dim=0) + smallest(dtype))
    status_clean(cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, "silu"), (torch.float16, "gelu"), (torch.float32, "silu"),
                                       (torch.float32, "gelu"), (torch.float32, "gelu_tanh")])
@pytest.mark.parametrize("m,n,k", GRAD_SHAPES)
@pytest.mark.parametrize("frozen", [False, True])
def test_gated_gradients(cuda_device, dtype, act, m, n, k, frozen):
    x, w1, b1 = make(m, n, k, dtype, m + 3 * n, cuda_device, bias=True)
    _x, w2, b2 = make(m, n, k, dtype, m + 3 * n + 1, cuda_device, bias=True)
    g = torch.Generator(device=cuda_device).manual_seed(11)
    dh = torch.randn((m, n), generator=g, device=cuda_device).to(dtype)
    ref = gated_reference(x, w1, w2, b1, b2, act)
    for t in (x, b1, b2) + (() if frozen else (w1, w2)):
        t.requires_grad_()
    if frozen:
        h = int8.int8_gated(x, int8.Int8Weight.from_float(w1), int8.Int8Weight.from_float(w2), b1, b2, activation=act)
        dx, db1, db2 = torch.autograd.grad(h, (x, b1, b2), dh)
    else:
        h = int8.int8_gated(x, w1, w2, b1, b2, activation=act)
        dx, dw1, dw2, db1, db2 = torch.autograd.grad(h, (x, w1, w2, b1, b2), dh)
    d64 = dh.double()
    d = [d64 * ref["u"] * ref["da"], d64 * ref["a"]]
    # error of D itself: the slack of the activation (its derivative: twice that), the error of u
    err = [d64.abs() * (act_slack(ref, 2.0) * ref["u"].abs() + 8 * U32 * 1.13 * ref["um"]) + 4 * U32 * d[0].abs(),
           d64.abs() * act_slack(ref) + 4 * U32 * d[1].abs()]
    both = torch.cat(d, 1)
    codes = torch.cat([ref["q1"], ref["q2"]], 0)
    scales = torch.cat([ref["t1"], ref["t2"]])
    want = (both * scales) @ codes
    assert_within(dx, want, grad_bound(both, torch.cat(err, 1), scales, codes, digit_limit(dtype), dtype, want))
    for i, db in enumerate((db1, db2)):
        want = d[i].sum(dim=0)
        assert_within(db, want, half_step(dtype) * want.abs() + (m + 2) * U32 * d[i].abs().sum(dim=0) + err[i].sum(dim=0) +
                      smallest(dtype))
    if not frozen:
        for i, dw in enumerate((dw1, dw2)):
            want = (d[i] * ref["s"][:, None]).T @ ref["q"]
            assert_within(dw, want, grad_bound(d[i].T, err[i].T, ref["s"], ref["q"], digit_limit(dtype), dtype, want))
    status_clean(cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
def test_gated_gradient_against_differences(cuda_device, act):
    """dx and dW against central differences, in 64 bits, of the block at the dequantised activations
    and weights (the point at which the straight-through gradient is the exact derivative)."""
    m, n, k = 6, 40, 24
    x, w1, b1 = make(m, n, k, torch.float32, 1, cuda_device, bias=True)
    _x, w2, b2 = make(m, n, k, torch.float32, 2, cuda_device, bias=True)
    for t in (x, w1, w2, b1, b2):
        t.requires_grad_()
    g = torch.Generator(device=cuda_device).manual_seed(3)
    dh = torch.randn((m, n), generator=g, device=cuda_device)
    grads = torch.autograd.grad(int8.int8_gated(x, w1, w2, b1, b2, activation=act), (x, w1, w2, b1, b2), dh)
    ref = gated_reference(x, w1, w2, b1, b2, act)
    point = [ref["q"] * ref["s"][:, None], ref["q1"] * ref["t1"][:, None], ref["q2"] * ref["t2"][:, None],
             b1.detach().double(), b2.detach().double()]

    def loss(xh, g1, g2, c1, c2):
        a, _ = plain_act(xh @ g1.T + c1, act)
        return (a * (xh @ g2.T + c2) * dh.double()).sum()

    for i, grad in enumerate(grads):
        v = torch.randn(point[i].shape, generator=g, device=cuda_device).double()
        eps = 1e-5
        hi = loss(*[p + eps * v if j == i else p for j, p in enumerate(point)])
        lo = loss(*[p - eps * v if j == i else p for j, p in enumerate(point)])
        slope = float((hi - lo) / (2 * eps))
        got = float((grad.double() * v).sum())
        size = float((grad.double() * v).abs().sum())
        # fp32 gradients (64 units of 2^-23 per summand at most), differences of order eps^2
        assert abs(got - slope) <= 1e-5 * size + 1e-7


@pytest.mark.gpu
def test_gradients_of_expanded_and_shared_tensors(cuda_device):
    """A summed loss hands down an expanded gradient; a weight and an activation used twice sum up."""
    m, n, k = 37, 50, 70
    x, w, _ = make(m, n, k, torch.float32, 4, cuda_device)
    x.requires_grad_()
    w.requires_grad_()
    ones = torch.ones((m, n), device=cuda_device)
    once = torch.autograd.grad(int8.int8_linear(x, w), (x, w), ones)
    summed = torch.autograd.grad(int8.int8_linear(x, w).sum(), (x, w))
    assert all(torch.equal(a, b) for a, b in zip(once, summed))
    twice = torch.autograd.grad(int8.int8_linear(x, w).sum() + int8.int8_linear(x, w).sum(), (x, w))
    assert all(torch.equal(2 * a, b) for a, b in zip(once, twice))
    # one tensor as both weights of the block, a transposed gradient
    dh = torch.randn((n, m), device=cuda_device).t()
    shared = torch.autograd.grad(int8.int8_gated(x, w, w), w, dh)[0]
    w2 = w.detach().clone().requires_grad_()
    parts = torch.autograd.grad(int8.int8_gated(x, w, w2), (w, w2), dh)
    assert torch.equal(shared, parts[0] + parts[1])
    # an activation broadcast over a batch: its gradient is the sum
    x3 = x.detach()[None].expand(3, m, k).requires_grad_()
    y = int8.int8_linear(x3, w.detach())
    assert y.shape == (3, m, n)
    gx = torch.autograd.grad(y.sum(), x3)[0]
    assert gx.shape == (3, m, k) and all(torch.equal(gx[i], once[0]) for i in range(3))


@pytest.mark.gpu
def test_gradients_of_mixed_types(cuda_device):
    """bf16 activations against fp32 master weights: each gradient in its tensor's type."""
    m, n, k = 50, 70, 90
    x, _w, _ = make(m, n, k, torch.bfloat16, 5, cuda_device)
    _x, w, b = make(m, n, k, torch.float32, 6, cuda_device, bias=True)
    _x, w2, _ = make(m, n, k, torch.bfloat16, 7, cuda_device)
    b2 = b.detach().half()
    for t in (x, w, b, w2, b2):
        t.requires_grad_()
    dy = torch.randn((m, n), device=cuda_device).to(torch.bfloat16)
    got = torch.autograd.grad(int8.int8_linear(x, w, b), (x, w, b), dy)
    assert [g.dtype for g in got] == [torch.bfloat16, torch.float32, torch.float32]
    (q, s), (wq, t) = plain_codes(x), plain_codes(w)
    want = (dy.double() * s[:, None]).T @ q
    none = torch.zeros((n, m), dtype=torch.float64, device=cuda_device)
    assert_within(got[1], want, grad_bound(dy.double().T, none, s, q, 8355000.0, torch.float32, want))
    got = torch.autograd.grad(int8.int8_gated(x, w, w2, b, b2), (x, w, w2, b, b2), dy)
    assert [g.dtype for g in got] == [t.dtype for t in (x, w, w2, b, b2)]
    assert all(bool(torch.isfinite(g).all()) for g in got)
    # one frozen projection beside a trained one: the trained one's gradient alone
    up = int8.Int8Weight.from_float(w2)
    alone = torch.autograd.grad(int8.int8_gated(x, w, up, b, b2), (x, w), dy)
    assert torch.equal(alone[0], got[0]) and torch.equal(alone[1], got[1])
    alone = torch.autograd.grad(int8.int8_gated(x, int8.Int8Weight.from_float(w), w2, b, b2), w2, dy)[0]
    # (its types are all bf16: two digits where the pass above took three)
    ref = gated_reference(x, w, w2, b, b2, "silu")
    d, err = dy.double() * ref["a"], dy.double().abs() * act_slack(ref)
    want = (d * ref["s"][:, None]).T @ ref["q"]
    for digits, g in ((32639.0, alone), (8355000.0, got[2])):
        assert_within(g, want, grad_bound(d.T, err.T, ref["s"], ref["q"], digits, torch.bfloat16, want))


@pytest.mark.gpu
def test_gradient_rows_with_nan_and_zero_rows(cuda_device):
    m, n, k = 20, 48, 64
    x, w, _ = make(m, n, k, torch.float32, 6, cuda_device)
    x.requires_grad_()
    dy = torch.randn((m, n), device=cuda_device)
    dy[3] = 0.0
    dy[5, 7] = float("nan")
    dx = torch.autograd.grad(int8.int8_linear(x, int8.Int8Weight.from_float(w)), x, dy)[0]
    assert torch.isnan(dx[5]).all() and float(dx[3].abs().max()) == 0.0
    rest = [i for i in range(m) if i != 5]
    assert torch.isfinite(dx[rest]).all()
    status_clean(cuda_device)


@pytest.mark.gpu
def test_results_do_not_depend_on_the_run(cuda_device):
    x, w, b = make(700, 300, 1000, torch.bfloat16, 8, cuda_device, bias=True)
    for t in (x, w, b):
        t.requires_grad_()
    dy = torch.randn((700, 300), device=cuda_device).to(torch.bfloat16)
    first = None
    for _ in range(4):
        y = int8.int8_linear(x, w, b)
        out = [y, *torch.autograd.grad(y, (x, w, b), dy)]
        if first is not None:
            assert all(torch.equal(p, q) for p, q in zip(first, out))
        first = out


# ---------------------------------------------------------------------------
# streams, graphs
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 200])
def test_captured_and_replayed_calls_follow_their_inputs(cuda_device, m):
    n, k = 200, 320
    x, w, _ = make(m, n, k, torch.bfloat16, 12, cuda_device)
    _x, w2, _ = make(m, n, k, torch.bfloat16, 13, cuda_device)
    g, u, d = (int8.Int8Weight.from_float(t) for t in (w, w2, w.t()))
    g.transposed(), u.transposed()

    def step():
        h = int8.int8_gated(x, g, u)
        y = int8.int8_linear(h, d)
        q, s = int8.per_token_int8(x)
        dx, *_ = int8.int8_gated_backward(h, q, s, g, u, dx_dtype=torch.bfloat16)
        dxl, dwl, _ = int8.int8_linear_backward(h, q, s, g, dx_dtype=torch.bfloat16, dw_dtype=torch.bfloat16)
        return h, y, dx, dxl, dwl

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):            # two graphs of the same calls alive at once
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for seed in (21, 22):
        x.copy_(synthetic.student_t_activations(m, k, seed, device=cuda_device))
        want = step()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    status_clean(cuda_device)


@pytest.mark.gpu
def test_captured_training_step_and_live_eager_graphs(cuda_device):
    """A captured forward and backward pass; refused while an eager graph of the same leaves lives (its
    accumulation node belongs to another stream), fine once it is gone."""
    m, n, k = 40, 64, 96
    x, w, b = make(m, n, k, torch.float32, 31, cuda_device, bias=True)
    for t in (x, w, b):
        t.requires_grad_()
    dy = torch.randn((m, n), device=cuda_device)

    def step():
        return torch.autograd.grad(int8.int8_gated(x, w, w, b, None), (x, w, b), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    alive = int8.int8_linear(x, w, b)
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            int8.int8_gated(x, w, w, b, None)
    torch.autograd.grad(alive, (x, w, b), dy)   # the eager graph is unharmed
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        x.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, step()))
    status_clean(cuda_device)


@pytest.mark.gpu
def test_codes_edited_between_forward_and_backward_are_refused(cuda_device):
    x, w, _ = make(8, 16, 32, torch.float32, 32, cuda_device)
    x.requires_grad_()
    wt = int8.Int8Weight.from_float(w)
    y = int8.int8_linear(x, wt)
    wt.codes.zero_()
    with pytest.raises(RuntimeError, match="modified in place"):
        y.sum().backward()


@pytest.mark.gpu
def test_kept_transposed_codes_on_another_stream(cuda_device):
    """The transposed copy a first backward pass makes is waited for by a pass on another stream."""
    x, w, _ = make(64, 3584, 4096, torch.bfloat16, 33, cuda_device)
    dy = torch.randn((64, 3584), device=cuda_device).to(torch.bfloat16)
    q, s = int8.per_token_int8(x)
    fresh = int8.Int8Weight.from_float(w)
    want = int8.int8_linear_backward(dy, q, s, fresh, dx_dtype=torch.bfloat16, keep_transposed=False)[0]
    for _ in range(5):
        wt = int8.Int8Weight.from_float(w)
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            first = int8.int8_linear_backward(dy, q, s, wt, dx_dtype=torch.bfloat16)[0]
        with torch.cuda.stream(b):
            second = int8.int8_linear_backward(dy, q, s, wt, dx_dtype=torch.bfloat16)[0]
        torch.cuda.synchronize()
        assert torch.equal(first, want) and torch.equal(second, want)


@pytest.mark.gpu
def test_two_streams_at_once(cuda_device):
    x, w, _ = make(300, 500, 1024, torch.bfloat16, 14, cuda_device)
    wt = int8.Int8Weight.from_float(w)
    small = x[:2]
    want, want_small = int8.int8_linear(x, wt), int8.int8_linear(small, wt)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, (st, inp) in enumerate(zip(streams, (x, small))):
            with torch.cuda.stream(st):
                outs[i].append(int8.int8_linear(inp, wt))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in outs[0]) and all(torch.equal(y, want_small) for y in outs[1])
    status_clean(cuda_device)


@pytest.mark.gpu
def test_edited_codes_reach_the_transposed_copy(cuda_device):
    x, w, _ = make(30, 40, 64, torch.float32, 15, cuda_device)
    wt = int8.Int8Weight.from_float(w)
    x.requires_grad_()
    dy = torch.randn((30, 40), device=cuda_device)
    torch.autograd.grad(int8.int8_linear(x, wt), x, dy)
    wt.codes[3].zero_()
    fresh = int8.Int8Weight(wt.codes.clone(), wt.scale)
    a = torch.autograd.grad(int8.int8_linear(x, wt), x, dy)[0]
    b = torch.autograd.grad(int8.int8_linear(x, fresh), x, dy)[0]
    assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# the student kernel "int8": linears and gated blocks of a model together
# ---------------------------------------------------------------------------
class GatedBlock(torch.nn.Module):
    def __init__(self, hidden, inter, act, bias=False):
        super().__init__()
        self.gate_proj = torch.nn.Linear(hidden, inter, bias=bias)
        self.up_proj = torch.nn.Linear(hidden, inter, bias=bias)
        self.down_proj = torch.nn.Linear(inter, hidden, bias=bias)
        self.act_fn = act

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class Model(torch.nn.Module):
    def __init__(self, act, bias):
        super().__init__()
        self.inp = torch.nn.Linear(48, 96)
        self.mlp = GatedBlock(96, 200, act, bias)
        self.head = torch.nn.Linear(96, 33, bias=False)

    def forward(self, x):
        h = self.inp(x)
        return self.head(h + self.mlp(h))


@pytest.mark.gpu
@pytest.mark.parametrize("act", [torch.nn.SiLU(), torch.nn.GELU(), torch.nn.GELU(approximate="tanh"), torch.nn.ReLU()])
@pytest.mark.parametrize("tokens", [(1,), (2, 70)])
def test_int8_student_model(cuda_device, monkeypatch, act, tokens):
    monkeypatch.setattr(students, "STUDENT_KERNEL", "int8")
    torch.manual_seed(0)
    model = Model(act, bias=True).to(cuda_device)
    x = torch.randn((*tokens, 48), device=cuda_device)
    with torch.no_grad():
        exact = model(x)
    names = students._replace_int32_linears(model)
    assert names == ["inp", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj", "head"]
    assert all(not isinstance(m, torch.nn.Linear) for m in model.modules())
    fused = not isinstance(act, torch.nn.ReLU)
    assert isinstance(model.mlp, students.Int8GatedMLP) == fused
    with torch.inference_mode(), students._Int32KernelProbe() as probe:
        y = model(x)
    assert probe.count == 5
    # every layer adds at most half a step of 1/127 of its rows' maxima on both sides; through the five
    # layers here that stays a small fraction of the output
    assert float((y - exact).norm() / exact.norm()) < 0.05
    # the same call by call
    h = int8.int8_linear(x, model.inp.int8_weight(), model.inp.bias)
    mlp = model.mlp
    g, u = mlp.gate_proj, mlp.up_proj
    if fused:
        p = int8.int8_gated(h, g.int8_weight(), u.int8_weight(), g.bias, u.bias, activation=mlp.activation)
    else:
        p = torch.relu(g(h)) * u(h)
    z = int8.int8_linear(h + mlp.down_proj(p), model.head.int8_weight())
    assert torch.equal(z, y)
    # a copy of the model, also after a backward pass (which leaves the transposed codes with the weights)
    model(x.clone().requires_grad_()).sum().backward()
    twin = copy.deepcopy(model)
    with torch.inference_mode():
        assert torch.equal(twin(x), y)
    # gradients reach the input through the frozen model
    xg = x.clone().requires_grad_()
    model(xg).square().sum().backward()
    assert xg.grad.shape == x.shape and torch.isfinite(xg.grad).all() and float(xg.grad.abs().max()) > 0
    status_clean(cuda_device)


@pytest.mark.gpu
def test_int8_student_of_an_fp8_linear(cuda_device, monkeypatch):
    monkeypatch.setattr(students, "STUDENT_KERNEL", "int8")
    x, w, ws = synthetic.make_linear_inputs(0, 0, synthetic.LinearShape("gate_proj", 96, 160), tokens=16, device=cuda_device)
    lin = torch.nn.Linear(160, 96, bias=False).to(cuda_device)
    lin.weight = torch.nn.Parameter(w, requires_grad=False)
    lin.weight_scale = ws
    model = torch.nn.Sequential(lin)
    students._replace_int32_linears(model)
    wd = w.float() * ws
    assert torch.equal(model(x), int8.int8_linear(x, wd))


def test_gated_blocks_are_recognised_by_their_children_alone():
    assert students._gated_activation(GatedBlock(4, 8, torch.nn.SiLU())) == "silu"
    assert students._gated_activation(GatedBlock(4, 8, torch.nn.GELU())) == "gelu"
    assert students._gated_activation(GatedBlock(4, 8, torch.nn.GELU(approximate="tanh"))) == "gelu_tanh"
    assert students._gated_activation(GatedBlock(4, 8, torch.nn.ReLU())) is None
    assert students._gated_activation(torch.nn.Sequential(torch.nn.Linear(2, 2))) is None
    odd = GatedBlock(4, 8, torch.nn.SiLU())
    odd.norm = torch.nn.LayerNorm(4)
    assert students._gated_activation(odd) is None


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(3, 40, 256), (300, 12000, 256), (1000, 5000, 256)])
def test_wait_that_runs_out_is_reported_and_the_next_call_is_exact(cuda_device, m, n, k):
    """Both forms of the product (split, and tiled) give up on a wait that nothing ends, report it and
    return; the next call is exact.  Nothing faults: see test_failure_detection.py."""
    a = torch.randint(-128, 128, (m, k), device=cuda_device, dtype=torch.int8)
    b = torch.randint(-128, 128, (n, k), device=cuda_device, dtype=torch.int8)
    nat.device_status(cuda_device.index or 0, clear=True)
    nat.call("ima_set_gemm_wait_test", 50_000)   # 50 microseconds
    try:
        int8.int8_gemm(a, b)
        code, where, detail = nat.device_status(cuda_device.index or 0, clear=True)
    finally:
        nat.call("ima_set_gemm_wait_test", 0)
    assert (code, detail) == (nat.IMA_ERR_TIMEOUT, -2) and where in (6, 7)
    c, _ = int8.int8_gemm(a, b)
    assert torch.equal(c, int_product(a, b))
    status_clean(cuda_device)


# ---------------------------------------------------------------------------
# operands whose rows do not start on 16 bytes
# ---------------------------------------------------------------------------
def test_pack_rows_refusals():
    lib, bad = nat.lib(), nat.IMA_ERR_INVALID_ARGUMENT
    assert lib.ima_int8_pack_rows(None, 0, 0, None, None, 0, 0, None, 7, 16, None) == 0
    assert lib.ima_int8_pack_rows(17, 2, 7, 32, None, 0, 0, None, 0, 16, None) == 0
    assert lib.ima_int8_pack_rows(17, -1, 7, 32, None, 0, 0, None, 7, 16, None) == bad
    assert lib.ima_int8_pack_rows(17, 2, 7, 33, None, 0, 0, None, 7, 16, None) == bad      # destination off 16 bytes
    assert lib.ima_int8_pack_rows(17, 2, 6, 32, None, 0, 0, None, 7, 16, None) == bad      # rows overlap
    assert lib.ima_int8_pack_rows(17, 2, 17, 32, None, 0, 0, None, 17, 16, None) == bad    # narrower than its rows
    assert lib.ima_int8_pack_rows(17, 2, 7, 32, None, 0, 0, None, 7, 24, None) == bad
    assert lib.ima_int8_pack_rows(17, 2, 7, 32, None, 3, 7, 64, 7, 16, None) == bad


def _laid_out(t, layout):
    """t in another layout: the same values at odd addresses, odd row strides or other orders."""
    r, c = t.shape
    if layout.startswith("offset"):
        at = int(layout[6:])
        out = torch.zeros(r * c + at, dtype=t.dtype, device=t.device)[at:].view(r, c)
    elif layout == "rows":
        out = torch.zeros((r, c + 5), dtype=t.dtype, device=t.device)[:, 3:3 + c]
    elif layout == "turned":
        out = torch.zeros((c, r + 3), dtype=t.dtype, device=t.device)[:, 1:r + 1].t()
    elif layout == "every second":
        out = torch.zeros((r, 2 * c), dtype=t.dtype, device=t.device)[:, ::2]
    else:
        assert layout == "plain"
        out = torch.zeros_like(t)
    out.copy_(t)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("a_layout,b_layout", [("offset1", "plain"), ("plain", "offset2"), ("offset3", "rows"),
                                               ("rows", "turned"), ("turned", "offset8"), ("every second", "rows"),
                                               ("turned", "turned")])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 5, 3), (3, 2, 16), (2, 129, 17), (7, 40, 31), (130, 300, 1718),
                                   (260, 65, 4099)])
def test_packed_operands(cuda_device, m, n, k, a_layout, b_layout):
    g = torch.Generator(device=cuda_device).manual_seed(m + n + k)
    a = torch.randint(-128, 128, (m, k), generator=g, device=cuda_device, dtype=torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=g, device=cuda_device, dtype=torch.int8)
    c, _ = int8.int8_gemm(_laid_out(a, a_layout), _laid_out(b, b_layout))
    assert torch.equal(c.double(), a.double() @ b.double().t())
    w = int8.Int8Weight(_laid_out(b, b_layout), torch.ones(n, device=cuda_device))
    assert torch.equal(w.codes, b)


@pytest.mark.gpu
def test_packed_rows_of_one_value(cuda_device):
    a = torch.randint(-128, 128, (1, 37), device=cuda_device, dtype=torch.int8)
    b = torch.randint(-128, 128, (4, 1), device=cuda_device, dtype=torch.int8)
    c, _ = int8.int8_gemm(a.expand(9, 37), b.expand(4, 37))
    assert torch.equal(c.double(), a.double().expand(9, 37) @ b.double().expand(4, 37).t())
    one = torch.randint(-128, 128, (1, 1), device=cuda_device, dtype=torch.int8)
    c, _ = int8.int8_gemm(one.expand(5, 1), b)
    assert torch.equal(c.double(), one.double().expand(5, 1) @ b.double().t())


@pytest.mark.gpu
def test_packed_buffer_has_zeros_behind_its_rows(cuda_device):
    src = torch.randint(-128, 128, (6 * 21 + 1,), device=cuda_device, dtype=torch.int8)[1:].view(6, 21)
    dst = torch.full((8, 48), 77, dtype=torch.int8, device=cuda_device)
    int8._call(torch.device("cuda", torch.cuda.current_device()), "ima_int8_pack_rows", src.data_ptr(), 6, 21,
               dst.data_ptr(), None, 0, 0, None, 21, 48)
    assert torch.equal(dst[:6, :21], src)
    assert (dst[:6, 21:32] == 0).all() and (dst[:6, 32:] == 77).all() and (dst[6:] == 77).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,pad", [(300, 260, 200, 0), (300, 260, 200, 2), (300, 262, 200, 1), (300, 261, 200, 0),
                                       (40, 262, 2000, 0), (129, 33, 64, 3), (257, 1, 64, 0)])
def test_outputs_of_every_alignment(cuda_device, dtype, m, n, k, pad):
    g = torch.Generator(device=cuda_device).manual_seed(n + pad)
    a = torch.randint(-128, 128, (m, k), generator=g, device=cuda_device, dtype=torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=g, device=cuda_device, dtype=torch.int8)
    ones = torch.full((max(m, n),), 2.0**-6, device=cuda_device)
    c_big = torch.full((m + 1, n + pad), 77, dtype=torch.int32, device=cuda_device)
    y_big = torch.full((m + 1, n + pad), 77.0, dtype=dtype, device=cuda_device)
    int8.int8_gemm(a, b, x_scale=ones[:m], w_scale=ones[:n], c_out=c_big[:m, pad:], y_out=y_big[:m, pad:])
    want = int_product(a, b)
    assert torch.equal(c_big[:m, pad:], want)
    assert torch.equal(y_big[:m, pad:], (want.float() * 2.0**-12).to(dtype))
    assert (c_big[m:] == 77).all() and (y_big[m:] == 77).all()
    assert (c_big[:, :pad] == 77).all() and (y_big[:, :pad] == 77).all()
    status_clean(cuda_device)


@pytest.mark.gpu
def test_empty_contraction_reads_no_stale_memory(cuda_device):
    """Scales of weights without columns are those of zeros, whatever lay in their memory."""
    for _ in range(4):
        for n in (5, 300):
            poison = [torch.full((n,), float("nan"), device=cuda_device) for _ in range(8)]
            del poison
            x, w = torch.randn((3, 0), device=cuda_device), torch.randn((n, 0), device=cuda_device)
            b = torch.randn((n,), device=cuda_device)
            for leaf in (x, w):
                leaf.requires_grad_()
            assert torch.equal(int8.int8_linear(x, w, b), b.expand(3, n))
            assert float(int8.int8_gated(x, w, w, b, None).detach().abs().sum()) == 0.0
            assert torch.equal(int8.int8_linear(x.detach(), w.detach(), b), b.expand(3, n))
            assert float(int8.int8_gated(x.detach(), w.detach(), w.detach(), b, None).abs().sum()) == 0.0
    status_clean(cuda_device)


@pytest.mark.gpu
def test_codes_without_columns_as_they_come(cuda_device):
    q = torch.empty((4, 0), dtype=torch.int8, device=cuda_device)
    w = int8.Int8Weight(torch.empty((3, 0), dtype=torch.int8, device=cuda_device), torch.ones(3, device=cuda_device))
    c, _ = int8.int8_gemm(q, w.codes)
    assert c.shape == (4, 3) and not c.any()
    dy = torch.ones((4, 3), device=cuda_device)
    dx, _dw, db = int8.int8_linear_backward(dy, q, torch.ones(4, device=cuda_device), w, dx_dtype=torch.float32,
                                            db_dtype=torch.float32)
    assert dx.shape == (4, 0) and torch.equal(db, torch.full((3,), 4.0, device=cuda_device))
    status_clean(cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
def test_scales_edited_between_forward_and_backward_are_refused(cuda_device, gated):
    x, w, _ = make(8, 16, 32, torch.float32, 33, cuda_device)
    x.requires_grad_()
    wt, up = int8.Int8Weight.from_float(w), int8.Int8Weight.from_float(w)
    y = int8.int8_gated(x, wt, up) if gated else int8.int8_linear(x, wt)
    (up if gated else wt).scale.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified in place"):
        y.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 8), (3, 9), (5, 1), (4, 1025), (2, 4100), (2, 21003), (1300, 1100), (1300, 4093),
                                 (1300, 5001), (1300, 10001)])
def test_quantiser_rows_at_every_alignment(cuda_device, dtype, m, k):
    g = torch.Generator(device=cuda_device).manual_seed(k)
    for at in range(1, 16 // dtype.itemsize + 1):
        flat = torch.randn((m * (k + at % 3) + at,), generator=g, device=cuda_device).to(dtype)
        x = flat[at:].view(m, k + at % 3)[:, :k]
        q, s = int8.per_token_int8(x)
        want_q, want_s = plain_codes(x)
        assert torch.equal(s.flatten().double(), want_s) and torch.equal(q.double(), want_q)
    status_clean(cuda_device)


@pytest.mark.gpu
def test_weights_of_other_ranks_are_refused(cuda_device):
    x = torch.randn((4, 32), device=cuda_device)
    for w in (torch.randn(32, device=cuda_device), torch.randn((2, 3, 32), device=cuda_device)):
        for grad in (False, True):
            w.requires_grad_(grad)
            with pytest.raises(RuntimeError, match="2-D"):
                int8.int8_linear(x, w)
            with pytest.raises(RuntimeError, match="2-D"):
                int8.int8_gated(x, w, w)
    status_clean(cuda_device)
