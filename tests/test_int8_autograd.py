"""What the int8 operators do under autograd beyond the plain backward pass."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from int_model_approximation_b200 import int8, students
from test_int8 import (U32, assert_within, digit_limit, grad_bound, half_step, make, plain_act, plain_codes, smallest,
                       status_clean)


# ---------------------------------------------------------------------------
# forward-mode tangents
# ---------------------------------------------------------------------------
def test_tangents_are_seen():
    t = torch.ones(3)
    int8._refuse_tangents(t, None)
    with forward_ad.dual_level():
        int8._refuse_tangents(t, None)
        with pytest.raises(RuntimeError, match="forward-mode"):
            int8._refuse_tangents(None, forward_ad.make_dual(t, t))


@pytest.mark.gpu
@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(cuda_device, requires_grad):
    x, w, b = make(4, 8, 32, torch.float32, 61, cuda_device, bias=True)
    wt = int8.Int8Weight.from_float(w)
    x.requires_grad_(requires_grad)
    with forward_ad.dual_level():
        dual, dual_bias = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(b, torch.ones_like(b))
        calls = [lambda: int8.int8_linear(dual, wt), lambda: int8.int8_linear(x, wt, dual_bias),
                 lambda: int8.int8_linear(x, forward_ad.make_dual(w, w)), lambda: int8.int8_gated(dual, wt, wt),
                 lambda: int8.int8_gated(x, wt, wt, None, dual_bias)]
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        y = int8.int8_linear(x, wt)
    assert torch.equal(y, int8.int8_linear(x, wt))
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda t: int8.int8_linear(t, wt), (x.detach(),), (torch.ones_like(x),))
    status_clean(cuda_device)


# ---------------------------------------------------------------------------
# linears wider than one exact contraction
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n", [0, 1, 17, int8.MAX_K - 1, int8.MAX_K, int8.MAX_K + 1, 152064, 262111, 262112, 262113, 393217,
                               1_000_003])
def test_parts_cover_the_contraction(n):
    parts = int8._parts(n)
    assert sum(count for _, count in parts) == n and all(0 <= count <= int8.MAX_K for _, count in parts)
    ends = [0]
    for first, count in parts:
        assert first == ends[-1] and first % 16 == 0 and (count > 0 or n == 0)
        ends.append(first + count)
    assert parts[0][1] == max(count for _, count in parts)
    assert (len(parts) == 1) == (n <= int8.MAX_K)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 131072, 64), (3, 131075, 33), (40, 152064, 96), (130, 262150, 48), (2, 131071, 32)])
@pytest.mark.parametrize("frozen", [False, True])
def test_gradients_of_a_vocabulary_head(cuda_device, dtype, m, n, k, frozen):
    x, w, b = make(m, n, k, dtype, 62, cuda_device, bias=True)
    g = torch.Generator(device=cuda_device).manual_seed(63)
    dy = torch.randn((m, n), generator=g, device=cuda_device)
    dy[:, n // 2:] *= 2.0**-6         # parts of different sizes
    dy = dy.to(dtype)
    (q, s), (wq, t) = plain_codes(x), plain_codes(w)
    for leaf in (x, b) if frozen else (x, w, b):
        leaf.requires_grad_()
    if frozen:
        y = int8.int8_linear(x, int8.Int8Weight.from_float(w), b)
        (dx, db), dw = torch.autograd.grad(y, (x, b), dy), None
    else:
        y = int8.int8_linear(x, w, b)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    want = (dy.double() * t) @ wq
    none = torch.zeros((m, n), dtype=torch.float64, device=cuda_device)
    # the parts' sums, each rounded to fp32, and their addition: within the six roundings of the bound
    assert_within(dx, want, grad_bound(dy.double(), none, t, wq, digit_limit(dtype), dtype, want))
    assert dx.dtype == dtype and db.dtype == dtype
    want = dy.double().sum(dim=0)
    assert_within(db, want, half_step(dtype) * want.abs() + (m + 2) * U32 * dy.double().abs().sum(dim=0) + smallest(dtype))
    if dw is not None:
        want = (dy.double() * s[:, None]).T @ q
        none = torch.zeros((n, m), dtype=torch.float64, device=cuda_device)
        assert_within(dw, want, grad_bound(dy.double().T, none, s, q, digit_limit(dtype), dtype, want))
    # the plain call, without and with kept transposed codes, gives the same
    wt = int8.Int8Weight.from_float(w)
    codes, scale = int8.per_token_int8(x)
    for keep in (False, True, True):
        got = int8.int8_linear_backward(dy, codes, scale, wt, dx_dtype=dtype, keep_transposed=keep)[0]
        assert torch.equal(got, dx) or not frozen
    status_clean(cuda_device)


@pytest.mark.gpu
def test_gradients_reach_the_input_of_a_model_with_a_wide_head(cuda_device, monkeypatch):
    monkeypatch.setattr(students, "STUDENT_KERNEL", "int8")
    torch.manual_seed(3)
    model = torch.nn.Sequential(torch.nn.Linear(64, 48), torch.nn.Linear(48, 131200, bias=False)).to(cuda_device)
    students._replace_int32_linears(model)
    x = torch.randn((7, 64), device=cuda_device, requires_grad=True)
    loss = torch.nn.functional.cross_entropy(model(x), torch.arange(7, device=cuda_device) * 18000)
    loss.backward()
    assert torch.isfinite(x.grad).all() and float(x.grad.abs().max()) > 0
    status_clean(cuda_device)


# ---------------------------------------------------------------------------
# digits of gradients over long sums
# ---------------------------------------------------------------------------
def test_digits_follow_types_and_lengths():
    b, h, f = torch.bfloat16, torch.float16, torch.float32
    assert int8._digit_count(1, b) == int8._digit_count(65536, b, None, b) == 2
    assert int8._digit_count(65537, b, b, None) == int8._digit_count(1, b, f) == int8._digit_count(1, h) == 3
    # the worst case of two digits over the longest sum that gets them is 0.6 of bf16's half step
    assert (65536 / 3) ** 0.5 * 2.0**-16 <= 0.6 * torch.finfo(b).eps / 2


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [70000, 131071])
@pytest.mark.parametrize("gated", [False, True])
def test_weight_gradient_that_one_token_carries(cuda_device, tokens, gated):
    """One token 2^14 times the others: the digits' error e is spread over all tokens, the result's norm is
    the one's.  A value that is off by e rounds to another bf16 number with probability e / step, and is then a step
    (2^-7 of it at most) off: sqrt(e 2^-7) of the norm.  Three digits: e <= sqrt(131071 / 3) 2^-24 < 2^-16, below
    2^-11 of the norm; with two it would be 5e-3."""
    n, k = 64, 96
    g = torch.Generator(device=cuda_device).manual_seed(64)
    x = torch.randn((tokens, k), generator=g, device=cuda_device).to(torch.bfloat16)
    w = (torch.randn((n, k), generator=g, device=cuda_device) * 0.05).to(torch.bfloat16).requires_grad_()
    dy = torch.randn((tokens, n), generator=g, device=cuda_device) * 2.0**-14
    dy[0] = torch.where(dy[0] < 0, -1.0, 1.0)
    dy = dy.to(torch.bfloat16)
    q, s = plain_codes(x)
    if gated:       # up at the constant bias 1, so that the gate's gradient is dy act'(g)
        up, one = torch.zeros((n, k), device=cuda_device), torch.ones(n, device=cuda_device)
        got, = torch.autograd.grad(int8.int8_gated(x, w, up, None, one), w, dy)
        wq, t = plain_codes(w)
        d = dy.double() * plain_act((q @ wq.T) * s[:, None] * t, "silu")[1]
    else:
        got, = torch.autograd.grad(int8.int8_linear(x, w), w, dy)
        d = dy.double()
    want = (d * s[:, None]).T @ q
    assert float((got.double() - want.to(torch.bfloat16).double()).norm()) <= 2.0**-10 * float(want.norm())
    status_clean(cuda_device)


def test_other_numbers_of_digits_are_refused():
    x, w = torch.zeros(2, 16), torch.zeros(4, 16)
    for digits in (0, 1, 4, 2.5, "2"):
        with pytest.raises(RuntimeError, match="2 or 3 digits"):
            int8.int8_linear(x, w, digits=digits)
        with pytest.raises(RuntimeError, match="2 or 3 digits"):
            int8.int8_gated(x, w, w, digits=digits)
        with pytest.raises(RuntimeError, match="2 or 3 digits"):
            int8.int8_linear_backward(x, x, x, w, digits=digits)
        with pytest.raises(RuntimeError, match="2 or 3 digits"):
            int8.int8_gated_backward(x, x, x, w, w, digits=digits)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,digits", [(torch.bfloat16, 2), (torch.bfloat16, 3), (torch.float32, 2), (torch.float32, 3)])
@pytest.mark.parametrize("m,n,k", [(3, 70, 33), (300, 130, 250)])
def test_wanted_digits(cuda_device, dtype, digits, m, n, k):
    """Every gradient within the digits that were asked for; a small token beside one of 2^18 times its size is kept
    by three digits and lost by two."""
    limit = {2: 32639.0, 3: 8355000.0}[digits]
    x, w, b = make(m, n, k, dtype, 65, cuda_device, bias=True)
    g = torch.Generator(device=cuda_device).manual_seed(66)
    dy = torch.randn((m, n), generator=g, device=cuda_device)
    dy[0] = torch.where(dy[0] < 0, -1.0, 1.0)
    dy[1:] = dy[1:].clamp(-1, 1) * 2.0**-18
    dy = dy.to(dtype)
    x.detach()[0, 1:] = 0     # the large token reaches one column of dW only; the scales stay alike
    x.detach()[0, 0] = 4.0
    for t in (x, w, b):
        t.requires_grad_()
    (q, s), (wq, t) = plain_codes(x), plain_codes(w)
    dx, dw, _ = torch.autograd.grad(int8.int8_linear(x, w, b, digits=digits), (x, w, b), dy)
    want = (dy.double() * t) @ wq
    none = torch.zeros((m, n), dtype=torch.float64, device=cuda_device)
    assert_within(dx, want, grad_bound(dy.double(), none, t, wq, limit, dtype, want))
    want = (dy.double() * s[:, None]).T @ q
    assert_within(dw, want, grad_bound(dy.double().T, none.T, s, q, limit, dtype, want))
    small = (dw.double()[:, 1:] - want[:, 1:]).norm() / want[:, 1:].norm()
    assert (float(small) < 0.2) == (digits == 3)
    codes, scale = int8.per_token_int8(x)
    got = int8.int8_linear_backward(dy, codes, scale, int8.Int8Weight.from_float(w), dx_dtype=dtype, dw_dtype=dtype,
                                    digits=digits)
    assert torch.equal(got[0], dx) and torch.equal(got[1], dw)
    # the gated block: the same digits through autograd and the plain call, and three closer than two
    h = int8.int8_gated(x, w, w, b, None, digits=digits)
    dx, dw = torch.autograd.grad(h, (x, w), dy)
    wt = int8.Int8Weight.from_float(w)
    got = int8.int8_gated_backward(dy, codes, scale, wt, wt, b, None, dx_dtype=dtype, dgate_dtype=dtype, dup_dtype=dtype,
                                   digits=digits)
    assert torch.equal(got[0], dx)
    status_clean(cuda_device)


# ---------------------------------------------------------------------------
# bias gradients
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n", [(2, 33), (129, 64), (1000, 70), (4096, 130)])
def test_bias_gradient_of_sums_that_cancel(cuda_device, dtype, m, n):
    """Pairs of rows of 2^10 and their negatives around rows of size 1: the 64-bit sums are off by m 2^-53 of the
    magnitudes, then rounded once."""
    g = torch.Generator(device=cuda_device).manual_seed(67)
    dy = torch.randn((m, n), generator=g, device=cuda_device)
    big = torch.randn((m // 2, n), generator=g, device=cuda_device) * 2.0**10
    dy[: m // 2] += big
    dy = dy.to(dtype)
    dy[m // 2 : m // 2 * 2] -= dy[: m // 2].flip(0)
    x, w, b = make(m, n, 32, dtype, 68, cuda_device, bias=True)
    b.requires_grad_()
    got, = torch.autograd.grad(int8.int8_linear(x, int8.Int8Weight.from_float(w), b), b, dy)
    want = dy.double().sum(dim=0)
    assert_within(got, want, half_step(dtype) * want.abs() + m * 2.0**-52 * dy.double().abs().sum(dim=0) + smallest(dtype))
    status_clean(cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [65536, 65537, 70000, 140000])
@pytest.mark.parametrize("digits", [None, 2, 3])
def test_long_sums_of_two_digits_come_in_parts(cuda_device, n, digits):
    """One channel that carries dx.  See test_weight_gradient_that_one_token_carries: three digits are off by less
    than 2^-10 of the norm behind bf16's own rounding, two by sqrt(sqrt(65536 / 3) 2^-16 2^-7), 2^-7.8, where a part is
    no longer than 65,536 and by sqrt(sqrt(131071 / 3) 2^-16 2^-7), 2^-7.6, where it is."""
    m, k = 5, 64
    x, w, _ = make(m, n, k, torch.bfloat16, 69, cuda_device)
    w[0] = torch.randn((k,), device=cuda_device).to(torch.bfloat16)
    g = torch.Generator(device=cuda_device).manual_seed(70)
    dy = torch.randn((m, n), generator=g, device=cuda_device) * 2.0**-12
    dy[:, 0] = 1.0
    dy = dy.to(torch.bfloat16)
    x.requires_grad_()
    wt = int8.Int8Weight.from_float(w)
    got, = torch.autograd.grad(int8.int8_linear(x, wt, digits=digits), x, dy)
    wq, t = plain_codes(w)
    want = (dy.double() * t) @ wq
    none = torch.zeros((m, n), dtype=torch.float64, device=cuda_device)
    limit = 8355000.0 if digits == 3 else 32639.0
    assert_within(got, want, grad_bound(dy.double(), none, t, wq, limit, torch.bfloat16, want))
    off = float((got.double() - want.to(torch.bfloat16).double()).norm() / want.norm())
    assert off <= (2.0**-10 if digits == 3 else 2.0**-7.8 if digits is None else 2.0**-7.6)
    status_clean(cuda_device)
