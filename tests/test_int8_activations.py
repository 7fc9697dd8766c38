"""The activations of the gated block by themselves: codes and scales are chosen so that g is a given fp32 number
exactly and u is 1, and h = act(g), the gate's bias gradient act'(g).

Bounds.  fp32 (steps of 2^-23, half of it per rounding): exp and the divisions by 1 to 2 are off by 2 steps
(their documented bounds), erfc by 4, every other operation by half a step: 8 steps, 16 half steps, of each term.  An
exponent or an erfc's argument that is itself rounded (gelu_tanh: z by 4 half steps; gelu: g / sqrt 2 and g^2 / 2 by 2)
carries |z| or g^2 + 2 times that into the value.  Below the smallest normal number each result is off by a
subnormal step 2^-149, which the factors beside it multiply.  Results of 16 bits take e^-|z| to 4 + |z| half steps more
(all that rounds to the type's own half step) and as 0 below 2^-126, |g| <= 88 times which is below 2^-119."""

from __future__ import annotations

import math

import pytest
import torch

from int_model_approximation_b200 import int8
from test_int8 import ACTS, U32, assert_within, half_step, smallest, status_clean

ROOT = math.sqrt(2.0 / math.pi)


def points(device):
    """fp32 numbers of both signs: around every sign change and extremum, along the tails, to both ends of the range."""
    tail = torch.linspace(0.0, 110.0, 1101, dtype=torch.float64)
    wide = torch.logspace(-45, 38.53, 400, dtype=torch.float64)
    near = torch.linspace(-3.0, 3.0, 1201, dtype=torch.float64)
    g = torch.cat([tail, -tail, wide, -wide, near]).float()
    return torch.cat([g, torch.tensor([3.4028234663852886e38, -3.4028234663852886e38])]).to(device)


def exact(g, act):
    """(value, slope, bounds of both) in 64 bits."""
    g = g.double()
    if act == "gelu":
        cdf, density = 0.5 * torch.erfc(-g / math.sqrt(2.0)), torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
        terms, grow = (cdf, g * density), 2.0 * (g * g + 2.0)
        value = g * cdf
    else:
        z, dz, grow = g, torch.ones_like(g), torch.zeros_like(g)
        if act == "gelu_tanh":
            z, dz = 2 * ROOT * (g + 0.044715 * g**3), 2 * ROOT * (1 + 3 * 0.044715 * g * g)
            grow = 4.0 * z.abs()
        r, c = torch.sigmoid(z), torch.sigmoid(-z)
        terms, value = (r, torch.where(c * r == 0, 0.0, g * r * c * dz)), g * r
    relative = torch.where(grow.isfinite() & (grow < 1e6), 16.0 + grow, 0.0) * U32   # far out both are 0 or exact
    tiny = 2.0**-149 * 8 * (1.0 + g.abs().clamp_max(128.0)) ** 3
    far = 4 * U32      # beyond: one multiplication and one addition
    value_bound = (relative + far) * value.abs() + tiny
    slope_bound = (relative + far) * (terms[0].abs() + terms[1].abs()) + tiny
    return value, terms[0] + terms[1], value_bound, slope_bound


def operands(g, dtype, tokens):
    """x, gate and up such that the product of gate is 1 * 1 * g and that of up is 1 * 1 * 1, exactly."""
    x = torch.zeros((tokens, 2), device=g.device, dtype=dtype)
    x[:, 0], x[:, 1] = 127.0, 1.0        # scale 1, codes 127 and 1
    codes = torch.zeros((g.numel(), 2), device=g.device, dtype=torch.int8)
    codes[:, 1] = 1
    return x, int8.Int8Weight(codes, g), int8.Int8Weight(codes.clone(), torch.ones_like(g))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [1, 33, 300])
def test_activation_of_given_numbers(cuda_device, act, dtype, tokens):
    g = points(cuda_device)
    if dtype == torch.float16:
        g = g.clamp(-60000.0, 60000.0)
    x, gate, up = operands(g, dtype, tokens)
    h = int8.int8_gated(x, gate, up, activation=act)
    want, _, bound, _ = exact(g, act)
    if dtype != torch.float32:
        z = 2 * ROOT * (g.double() + 0.044715 * g.double() ** 3) if act == "gelu_tanh" else g.double()
        relative = half_step(dtype) + (4 + z.abs().clamp_max(150.0)) * U32
        bound = bound + relative * want.abs() + 2.0**-119 + smallest(dtype)
    fits = want.abs() < torch.finfo(dtype).max * (1 - 2.0**-9)
    assert_within(h[0][fits], want[fits], bound[fits])
    assert not h.isnan().any() and all(torch.equal(row, h[0]) for row in h[1::37])
    status_clean(cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("tokens", [1, 33, 300])
def test_slope_of_given_numbers(cuda_device, act, tokens):
    g = points(cuda_device)
    x, gate, up = operands(g, torch.float32, tokens)
    bias = torch.zeros_like(g).requires_grad_()     # adds +0: g + 0 is g
    dh = torch.zeros((tokens, g.numel()), device=cuda_device)
    dh[tokens // 2] = 1.0                           # the other tokens add zeros
    got, = torch.autograd.grad(int8.int8_gated(x, gate, up, bias, None, activation=act), bias, dh)
    _, want, _, bound = exact(g, act)
    assert_within(got, want, bound)
    status_clean(cuda_device)
