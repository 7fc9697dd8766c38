"""Int8Weight handles over their lifetime: captures, edits, replaced tensors.  The CPU tests replace the
transposing launch and the stream queries by host ones; what the handle decides is the same."""

from __future__ import annotations

import pytest
import torch

from int_model_approximation_b200 import int8
from test_int8 import make, status_clean


class FakeStream:
    cuda_stream = 7


class FakeEvent:
    def record(self, stream):
        pass

    def query(self):
        return True


@pytest.fixture
def host_handle(monkeypatch):
    """An Int8Weight of host tensors, and a switch that says whether a capture runs."""
    stream, capturing = FakeStream(), [False]
    monkeypatch.setattr(int8, "_require_cuda", lambda *named: None)
    monkeypatch.setattr(int8.nat, "require_device", lambda *named: None)
    monkeypatch.setattr(int8, "_transpose", lambda t: t.t().contiguous())
    monkeypatch.setattr(int8, "_raw_stream", lambda index: stream.cuda_stream)
    monkeypatch.setattr(int8, "_capturing", lambda *index: capturing[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *device: stream)
    monkeypatch.setattr(torch.cuda, "Event", FakeEvent)
    wt = int8.Int8Weight.__new__(int8.Int8Weight)
    wt._set(torch.randint(-127, 128, (5, 16), dtype=torch.int8), torch.ones(5))
    return wt, capturing


def test_a_capture_takes_no_kept_transposed_codes(host_handle):
    wt, capturing = host_handle
    kept = wt.transposed()
    assert torch.equal(kept, wt.codes.t()) and wt.transposed() is kept
    capturing[0] = True
    assert wt.transposed() is None
    capturing[0] = False
    assert wt.transposed() is kept
    wt.codes[2].zero_()
    assert torch.equal(wt.transposed(), wt.codes.t())


@pytest.mark.gpu
@pytest.mark.parametrize("own_stream", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_replays_follow_edited_codes(cuda_device, own_stream, gated):
    """A backward pass captured while transposed copies are kept (made on the capturing stream, or on another one
    and complete), then the codes edited, an eager pass that renews the copies, and memory reused."""
    m, n, k = 40, 70, 200
    x, w, _ = make(m, n, k, torch.float32, 51, cuda_device)
    _x, w2, _ = make(m, n, k, torch.float32, 52, cuda_device)
    dy = torch.randn((m, n), device=cuda_device)
    q, s = int8.per_token_int8(x)
    g, u = int8.Int8Weight.from_float(w), int8.Int8Weight.from_float(w2)

    def step(g, u):
        if gated:
            return int8.int8_gated_backward(dy, q, s, g, u, dx_dtype=torch.float32)[0]
        return int8.int8_linear_backward(dy, q, s, g, dx_dtype=torch.float32)[0]

    capturing = torch.cuda.Stream()
    with torch.cuda.stream(capturing if own_stream else torch.cuda.current_stream()):
        step(g, u)
    torch.cuda.synchronize()
    with torch.cuda.stream(capturing):
        for _ in range(2):      # the copies are known to be complete here
            step(g, u)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=capturing):
        got = step(g, u)
    for wt in (g, u):
        wt.codes[3].zero_()
        wt.codes[:, 5].fill_(100)
    want = step(*(int8.Int8Weight(wt.codes.clone(), wt.scale) for wt in (g, u)))
    step(g, u)
    scribble = [torch.full((k, 80), 77, dtype=torch.int8, device=cuda_device) for _ in range(64)]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(step(g, u), want)
    del scribble
    status_clean(cuda_device)


# ---------------------------------------------------------------------------
# codes and scales that lie elsewhere than before
# ---------------------------------------------------------------------------
def test_repointed_codes_are_transposed_anew(host_handle):
    wt, _capturing = host_handle
    wt.transposed()
    version = wt.codes._version
    wt.codes.data = torch.randint(-127, 128, (5, 16), dtype=torch.int8)
    assert wt.codes._version == version       # the version alone does not tell
    assert torch.equal(wt.transposed(), wt.codes.t())


def test_codes_and_scales_are_not_assigned(host_handle):
    wt, _capturing = host_handle
    for name in ("codes", "scale"):
        with pytest.raises(AttributeError):
            setattr(wt, name, getattr(wt, name).clone())


@pytest.mark.gpu
def test_repointed_codes_and_scales(cuda_device):
    """tensor.data = other, of another shape too: forward and backward follow; between the two it is refused."""
    dev = cuda_device
    x, w, _ = make(9, 40, 64, torch.float32, 53, dev)
    _x, w2, _ = make(9, 130, 64, torch.float32, 54, dev)
    x.requires_grad_()
    dy, dy2 = torch.randn((9, 40), device=dev), torch.randn((9, 130), device=dev)
    wt = int8.Int8Weight.from_float(w)
    torch.autograd.grad(int8.int8_linear(x, wt), x, dy)
    other = int8.Int8Weight.from_float(w2)
    y = int8.int8_linear(x, wt)
    wt.codes.data, wt.scale.data = other.codes.clone(), other.scale.clone()
    with pytest.raises(RuntimeError, match="modified in place"):
        torch.autograd.grad(y, x, dy, retain_graph=True)
    y, want = int8.int8_linear(x, wt), int8.int8_linear(x, other)
    assert torch.equal(y, want)
    want, = torch.autograd.grad(want, x, dy2)
    assert torch.equal(torch.autograd.grad(y, x, dy2)[0], want)
    q, s = int8.per_token_int8(x)
    assert torch.equal(int8.int8_linear_backward(dy2, q, s, wt, dx_dtype=torch.float32)[0], want)
    h = int8.int8_gated(x.detach(), wt, other)
    assert torch.equal(h, int8.int8_gated(x.detach(), other, other))
    # back and forth: memory of the same address, other values
    wt = int8.Int8Weight.from_float(w)
    y = int8.int8_linear(x, wt)
    torch.autograd.grad(y, x, dy, retain_graph=True)
    for fill in (3, 5, 7):
        wt.codes.data = torch.full((40, 64), fill, dtype=torch.int8, device=dev)
        fresh = int8.Int8Weight(wt.codes.clone(), wt.scale.clone())
        z, want = int8.int8_linear(x, wt), int8.int8_linear(x, fresh)
        assert torch.equal(z, want)
        assert torch.equal(torch.autograd.grad(z, x, dy)[0], torch.autograd.grad(want, x, dy)[0])
        with pytest.raises(RuntimeError, match="modified in place"):
            torch.autograd.grad(y, x, dy, retain_graph=True)
    # the same memory, fewer rows
    wt.codes.data, wt.scale.data = wt.codes[:17], wt.scale[:17]
    assert int8.int8_linear(x, wt).shape == (9, 17)
    wt = int8.Int8Weight(other.codes.clone(), other.scale.clone())
    # layouts that the kernels cannot read
    wt.scale.data = torch.ones(7, device=dev)
    with pytest.raises(RuntimeError, match="entries, expected"):
        int8.int8_linear(x, wt)
    wt.scale.data = torch.ones(260, device=dev)[::2]
    with pytest.raises(RuntimeError, match="contiguous fp32"):
        int8.int8_linear(x, wt)
    wt.scale.data = other.scale.clone()
    wt.codes.data = torch.zeros((130, 65), dtype=torch.int8, device=dev)[:, 1:]
    with pytest.raises(RuntimeError, match="do not start on 16 bytes"):
        int8.int8_gated(x, wt, other)
    status_clean(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("gated,n", [(False, 70), (False, 131080), (True, 70)])
def test_replayed_training_steps_follow_edited_codes(cuda_device, gated, n):
    """Forward and backward through autograd, captured while transposed copies are kept; then codes and scales edited."""
    m, k = 20, 48
    x, w, _ = make(m, n, k, torch.float32, 55, cuda_device)
    x.requires_grad_()
    dy = torch.randn((m, n), device=cuda_device)
    wt = int8.Int8Weight.from_float(w)

    def step(wt):
        y = int8.int8_gated(x, wt, wt) if gated else int8.int8_linear(x, wt)
        return y.detach(), *torch.autograd.grad(y, x, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(wt)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(wt)
    for edit in (lambda: wt.codes[3].fill_(100), lambda: wt.scale.mul_(1.5), lambda: wt.codes[:, 1].zero_()):
        edit()
        graph.replay()
        torch.cuda.synchronize()
        want = step(int8.Int8Weight(wt.codes.clone(), wt.scale.clone()))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del want
    status_clean(cuda_device)
