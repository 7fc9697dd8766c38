"""Calls from threads that have made no CUDA call before: workers of a server, autograd's own thread."""

from __future__ import annotations

import os
import subprocess
import sys
import threading

import pytest
import torch

from int_model_approximation_b200 import codebook, int8
from test_int8 import make, status_clean


def in_new_thread(call):
    """call() as all that a new thread does; its result or exception."""
    out = {}

    def work():
        try:
            out["result"] = call()
        except BaseException as e:
            out["error"] = e

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    if "error" in out:
        raise out["error"]
    return out["result"]


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 300])
def test_first_calls_of_a_thread(cuda_device, m):
    x, w, b = make(m, 70, 96, torch.bfloat16, 71, cuda_device, bias=True)
    wt = int8.Int8Weight.from_float(w)
    q, s = int8.per_token_int8(x)
    dy = torch.randn((m, 70), device=cuda_device)
    bf = torch.bfloat16
    calls = [lambda: int8.int8_linear(x, wt, b), lambda: int8.int8_linear(x, w, b),
             lambda: int8.int8_gated(x, wt, wt, b), lambda: int8.per_token_int8(x)[0],
             lambda: int8.int8_gemm(q, wt.codes)[0],
             lambda: int8.int8_linear_backward(dy, q, s, wt, dx_dtype=bf)[0],
             lambda: int8.int8_linear_backward(dy, q, s, wt, db_dtype=bf)[2],
             lambda: int8.int8_gated_backward(dy, q, s, wt, wt, dx_dtype=bf)[0],
             lambda: int8.int8_gated_backward(dy, q, s, wt, wt, gate_db_dtype=bf)[3]]
    for call in calls:
        want = call()
        torch.cuda.synchronize()
        got = in_new_thread(call)
        assert torch.equal(got, want)
    status_clean(cuda_device)


@pytest.mark.gpu
def test_first_codebook_product_of_a_thread(cuda_device):
    a = torch.randint(-400, 400, (30, 64), dtype=torch.int32, device=cuda_device)
    b = torch.randint(-400, 400, (64, 50), dtype=torch.int32, device=cuda_device)
    planes = codebook.planes_from_int32(a), codebook.planes_from_int32(b, transpose=True)
    want = codebook.int_gemm(*planes)[0]
    torch.cuda.synchronize()
    assert torch.equal(in_new_thread(lambda: codebook.int_gemm(*planes)[0]), want)
    status_clean(cuda_device)


BIAS_ONLY = """
import torch
from int_model_approximation_b200 import int8
dev = torch.device("cuda", 0)
x, w = torch.randn((5, 64), device=dev), torch.randn((40, 64), device=dev)
wt = int8.Int8Weight.from_float(w)
bias = torch.zeros(40, device=dev, requires_grad=True)
int8.int8_gated(x, wt, wt, bias, None).sum().backward()     # the only gradient: no launch before the products
assert torch.isfinite(bias.grad).all() and float(bias.grad.abs().max()) > 0
print("ok")
"""


@pytest.mark.gpu
def test_first_call_of_the_autograd_thread(cuda_device):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", BIAS_ONLY], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stderr[-2000:]


@pytest.mark.gpu
def test_threads_at_once(cuda_device):
    """Four threads, a stream each, the same weight."""
    x, w, _ = make(64, 300, 512, torch.bfloat16, 72, cuda_device)
    wt = int8.Int8Weight.from_float(w)
    q, s = int8.per_token_int8(x)
    dy = torch.randn((64, 300), device=cuda_device).to(torch.bfloat16)
    want = int8.int8_linear(x, wt), int8.int8_linear_backward(dy, q, s, wt, dx_dtype=torch.bfloat16)[0]
    torch.cuda.synchronize()
    results, errors = [], []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream(cuda_device)):
                for _ in range(20):
                    results.append((int8.int8_linear(x, wt),
                                    int8.int8_linear_backward(dy, q, s, wt, dx_dtype=torch.bfloat16)[0]))
        except BaseException as e:
            errors.append(e)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors and len(results) == 80
    assert all(torch.equal(a, b) for pair in results for a, b in zip(pair, want))
    status_clean(cuda_device)
