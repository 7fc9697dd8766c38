"""The student kernel "int8": which modules it replaces, and by what."""

from __future__ import annotations

import pytest
import torch

from int_model_approximation_b200 import int8, students, synthetic
from test_int8 import GatedBlock, status_clean


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


# ---------------------------------------------------------------------------
# which modules are gated blocks
# ---------------------------------------------------------------------------
class Fp32Activation(GatedBlock):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x).float()).to(x.dtype) * self.up_proj(x))


class OtherOrder(GatedBlock):
    def forward(self, hidden_states):
        return self.down_proj(self.up_proj(hidden_states) * self.act_fn(self.gate_proj(hidden_states)))


class Clamped(GatedBlock):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x).clamp(max=7.0)) * self.up_proj(x))


class Shifted(GatedBlock):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * (self.up_proj(x) + 1))


class Scaled(GatedBlock):
    multiplier = 0.5

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x) * self.multiplier) * self.up_proj(x))


class Residual(GatedBlock):
    def forward(self, x):
        return x + self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class Swapped(GatedBlock):
    def forward(self, x):
        return self.down_proj(self.gate_proj(x) * self.act_fn(self.up_proj(x)))


class Dropping(GatedBlock):
    def forward(self, x):
        h = self.act_fn(self.gate_proj(x)) * self.up_proj(x)
        return self.down_proj(torch.nn.functional.dropout(h, 0.5, self.training))


class WithMask(GatedBlock):
    def forward(self, x, mask=None):
        h = self.act_fn(self.gate_proj(x)) * self.up_proj(x)
        return self.down_proj(h if mask is None else h * mask)


class Raising(GatedBlock):
    def forward(self, x):
        return self.down_proj(self.act_fn(x @ self.gate_proj.weight.t()) * self.up_proj(x))


ACT_MODULES = {"silu": torch.nn.SiLU(), "gelu": torch.nn.GELU(), "gelu_tanh": torch.nn.GELU(approximate="tanh")}


@pytest.mark.parametrize("act", sorted(ACT_MODULES))
@pytest.mark.parametrize("sizes", [(4, 8), (1, 3), (7, 5), (64, 200)])
def test_blocks_of_the_formula_are_recognised(act, sizes):
    for cls in (GatedBlock, Fp32Activation, OtherOrder):
        block = cls(*sizes, ACT_MODULES[act])
        before = torch.random.get_rng_state()
        assert students._gated_activation(block) == act
        assert students._gated_activation(block.double().eval()) == act
        assert torch.equal(before, torch.random.get_rng_state()) and isinstance(block.gate_proj, torch.nn.Linear)


@pytest.mark.parametrize("act", sorted(ACT_MODULES))
@pytest.mark.parametrize("cls", [Clamped, Shifted, Scaled, Residual, Swapped, Dropping, WithMask, Raising])
def test_blocks_of_another_formula_are_left_alone(cls, act):
    for block in (cls(16, 24, ACT_MODULES[act]), cls(16, 24, ACT_MODULES[act]).eval()):
        assert students._gated_activation(block) is None


def test_blocks_with_something_of_their_own_are_left_alone():
    block = GatedBlock(4, 8, torch.nn.SiLU())
    block.register_buffer("scale", torch.ones(1))
    assert students._gated_activation(block) is None
    block = GatedBlock(4, 8, torch.nn.SiLU())
    block.gain = torch.nn.Parameter(torch.ones(1))
    assert students._gated_activation(block) is None
    block = GatedBlock(4, 8, torch.nn.SiLU())
    block.forward = lambda x: GatedBlock.forward(block, x)
    assert students._gated_activation(block) is None

    class Leaky(torch.nn.SiLU):     # an activation of that class that computes another
        def forward(self, x):
            return torch.nn.functional.leaky_relu(x)

    assert students._gated_activation(GatedBlock(4, 8, Leaky())) is None
    for part in (None, "gate_proj", "up_proj", "act_fn"):
        for register in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook",
                         "register_full_backward_pre_hook"):
            block = GatedBlock(4, 8, torch.nn.SiLU())
            handle = getattr(block if part is None else getattr(block, part), register)(lambda *args: None)
            assert students._gated_activation(block) is None
            handle.remove()
            assert students._gated_activation(block) == "silu"


@pytest.mark.gpu
def test_students_of_other_blocks_compute_what_the_blocks_do(cuda_device, monkeypatch):
    """Through the replacement pass: fused or not, a block's student stays near the block."""
    monkeypatch.setattr(students, "STUDENT_KERNEL", "int8")
    torch.manual_seed(1)
    x = torch.randn((30, 64), device=cuda_device) * 4
    for cls in (GatedBlock, Fp32Activation, Clamped, Shifted, Scaled, Residual, Swapped, WithMask):
        model = torch.nn.Sequential(cls(64, 96, torch.nn.SiLU(), bias=True)).to(cuda_device).eval()
        with torch.no_grad():
            model[0].gate_proj.weight.mul_(4)   # gates beyond the clamp
            want = model(x)
            students._replace_int32_linears(model)
            got = model(x)
        assert isinstance(model[0], students.Int8GatedMLP) == (cls in (GatedBlock, Fp32Activation))
        # a percent or two from three linears of half a step of 1/127; every other formula is tens of percent off
        assert float((got - want).norm() / want.norm()) < 0.05, cls
    status_clean(cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("act", sorted(ACT_MODULES))
def test_hooks_on_the_projections_of_a_fused_block(cuda_device, monkeypatch, act):
    monkeypatch.setattr(students, "STUDENT_KERNEL", "int8")
    torch.manual_seed(2)
    model = torch.nn.Sequential(GatedBlock(64, 96, ACT_MODULES[act], bias=True)).to(cuda_device)
    students._replace_int32_linears(model)
    block = model[0]
    assert isinstance(block, students.Int8GatedMLP)
    x = torch.randn((5, 64), device=cuda_device, requires_grad=True)
    plain = model(x)
    seen = []
    handles = [block.gate_proj.register_forward_hook(lambda m, args, out: seen.append(out.detach())),
               block.up_proj.register_forward_pre_hook(lambda m, args: (args[0] * 2,)),
               block.down_proj.register_forward_hook(lambda m, args, out: seen.append(args[0].detach()))]
    with students._Int32KernelProbe() as probe:
        y = model(x)
    assert probe.count == 3 and len(seen) == 2
    g = int8.int8_linear(x, block.gate_proj.int8_weight(), block.gate_proj.bias).detach()
    u = int8.int8_linear(x * 2, block.up_proj.int8_weight(), block.up_proj.bias).detach()
    assert torch.equal(seen[0], g) and torch.equal(seen[1], ACT_MODULES[act](g) * u)
    grads = []
    handles.append(block.gate_proj.register_full_backward_hook(lambda m, gi, go: grads.append(go[0])))
    model(x).sum().backward()
    assert len(grads) == 1 and grads[0].shape == (5, 96)
    for handle in handles:
        handle.remove()
    assert torch.equal(model(x), plain) and not torch.equal(y, plain)
    status_clean(cuda_device)


# ---------------------------------------------------------------------------
# modules that are moved or cast
# ---------------------------------------------------------------------------
def host_linear(n=6, k=16, bias=True):
    """An Int8Linear of host tensors, without the launch that quantises."""
    made = students.Int8Linear.__new__(students.Int8Linear)
    torch.nn.Module.__init__(made)
    made.register_buffer("weight", torch.randint(-127, 128, (n, k), dtype=torch.int8), persistent=False)
    made.register_buffer("weight_scale", torch.logspace(-9, 2, n), persistent=False)
    made.register_buffer("bias", torch.randn(n), persistent=False)
    made.in_features, made.out_features = k, n
    return made


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_a_cast_leaves_the_scales_of_the_codes(dtype):
    lin = host_linear()
    codes, scale = lin.weight.clone(), lin.weight_scale.clone()
    model = torch.nn.Sequential(lin).to(dtype)
    assert model[0] is lin and lin.bias.dtype == dtype
    assert torch.equal(lin.weight, codes) and lin.weight_scale.dtype == torch.float32
    assert torch.equal(lin.weight_scale, scale)
    meta = model.to(device="meta", dtype=dtype)[0]
    assert meta.weight_scale.dtype == torch.float32 and meta.weight_scale.device.type == "meta"


@pytest.mark.gpu
def test_a_cast_model_computes_with_its_own_scales(cuda_device):
    w = torch.randn((40, 64), device=cuda_device) * torch.logspace(-9, 0, 40, device=cuda_device)[:, None]
    lin = students.Int8Linear(w, None)
    x = torch.randn((3, 64), device=cuda_device).to(torch.float16)
    want = int8.int8_linear(x, int8.Int8Weight.from_float(w))
    for cast in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.float(), lambda m: m.cpu().to(cuda_device)):
        lin = cast(lin)
        assert torch.equal(lin(x), want)
    status_clean(cuda_device)


# ---------------------------------------------------------------------------
# activations of other classes
# ---------------------------------------------------------------------------
class OwnGelu(torch.nn.Module):
    def forward(self, x):
        return 0.5 * x * (1.0 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x**3)))


class OwnSilu(torch.nn.Module):
    def forward(self, x):
        return x * torch.sigmoid(x)


class ScaledSilu(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.beta = torch.nn.Parameter(torch.ones(1))

    def forward(self, x):
        return x * torch.sigmoid(self.beta * x)


def test_activations_of_other_classes():
    assert students._gated_activation(GatedBlock(4, 8, OwnGelu())) == "gelu_tanh"
    assert students._gated_activation(GatedBlock(4, 8, OwnSilu())) == "silu"
    assert students._gated_activation(GatedBlock(4, 8, torch.nn.Sequential(torch.nn.SiLU()))) == "silu"
    quick = torch.nn.Module()
    quick.forward = lambda x: x * torch.sigmoid(1.702 * x)
    dropping = torch.nn.Sequential(torch.nn.SiLU(), torch.nn.Dropout(0.5))
    for act in (ScaledSilu(), quick, dropping, dropping.eval(), torch.nn.Mish(), torch.nn.Tanh(), torch.nn.Identity()):
        assert students._gated_activation(GatedBlock(4, 8, act)) is None
    hooked = torch.nn.Sequential(torch.nn.SiLU())
    hooked[0].register_forward_hook(lambda *args: None)
    assert students._gated_activation(GatedBlock(4, 8, hooked)) is None
