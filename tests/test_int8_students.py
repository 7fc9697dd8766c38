"""The student kernel "int8": which modules it replaces, and by what."""

from __future__ import annotations

import pytest
import torch

from int_model_approximation_b200 import int8, students, synthetic
from test_int8 import status_clean


def fp8_linear(n, k, scale, seed=0, device="cpu"):
    w, _ = synthetic.normal_fp8_weights(n, k, seed=seed)
    lin = torch.nn.Linear(k, n, bias=False, device=device)
    lin.weight = torch.nn.Parameter(w.to(device), requires_grad=False)
    lin.weight_scale = scale.to(device)
    return lin


# ---------------------------------------------------------------------------
# scales of FP8 linears
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n,k", [(6, 6), (6, 4), (1, 5)])
@pytest.mark.parametrize("shape", [(-1,), (-1, 1), (1, -1)])
def test_fp8_channel_scales_of_any_shape(n, k, shape):
    scale = torch.linspace(0.5, 2.0, n)
    got = students._dequantized_weight(fp8_linear(n, k, scale.reshape(shape)))
    w, _ = synthetic.normal_fp8_weights(n, k, seed=0)
    assert torch.equal(got, w.float() * scale[:, None])


def test_fp8_scales_of_a_whole_weight_and_of_other_shapes():
    w, _ = synthetic.normal_fp8_weights(6, 4, seed=0)
    for scale in (torch.tensor(0.25), torch.tensor([0.25]), torch.tensor([[0.25]])):
        assert torch.equal(students._dequantized_weight(fp8_linear(6, 4, scale)), w.float() * 0.25)
    for scale in (torch.ones(4), torch.ones(1, 4), torch.ones(3, 2, 2), torch.ones(0)):
        with pytest.raises(RuntimeError, match="weight_scale"):
            students._dequantized_weight(fp8_linear(6, 4, scale))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(-1,), (-1, 1)])
def test_square_fp8_linear_beside_the_codebook_student(cuda_device, monkeypatch, shape):
    """Scales that differ by 64 between channels: along the wrong side they would be far off the codebook's output."""
    n = 96
    scale = torch.logspace(-2, 4, n, base=2.0).reshape(shape)
    lin = fp8_linear(n, n, scale, seed=3, device=cuda_device)
    x = synthetic.student_t_activations(20, n, 4, device=cuda_device)
    with torch.no_grad():
        want = students.CodebookLinear(lin.weight, lin.weight_scale, None)(x).float()
    monkeypatch.setattr(students, "STUDENT_KERNEL", "int8")
    model = torch.nn.Sequential(lin)
    students._replace_int32_linears(model)
    with torch.no_grad():
        got = model(x).float()
        assert torch.equal(model(x), int8.int8_linear(x, lin.weight.float() * scale.to(cuda_device).reshape(-1, 1)))
    # e4m3 carries 2^-4 of each activation, int8 half a step of 1/127 of the row's maximum
    assert float((got - want).norm() / want.norm()) < 0.1
    status_clean(cuda_device)
