"""GPU: calls from threads that have not used CUDA yet. A new thread has no CUDA context bound, and torch
binds none while its allocator serves from its cache, so a call's tensor maps can be the thread's first
use of the driver."""

from __future__ import annotations

import subprocess
import sys
import threading

import pytest
import torch

from diffucore_b200 import _lib, kernels, text
from tests.conftest import ROOT

pytestmark = pytest.mark.gpu
DEV = "cuda"


def in_fresh_thread(call):
    """``call`` once here, so that the allocator's cache has its blocks, then in a new thread."""
    want = call()
    got = []

    def run():
        try:
            got.append(call())
        except Exception as e:  # noqa: BLE001  handed to the test's thread
            got.append(e)

    torch.cuda.synchronize()
    thread = threading.Thread(target=run)
    thread.start()
    thread.join()
    if isinstance(got[0], Exception):
        raise got[0]
    torch.cuda.synchronize()
    assert torch.equal(got[0], want)


def rand(*shape):
    return torch.randn(*shape, device=DEV).to(torch.bfloat16)


def test_projections():
    x, w, dz = rand(300, 256), rand(512, 256), rand(300, 512)
    in_fresh_thread(lambda: text.linear(x, w))
    in_fresh_thread(lambda: text.gated_linear(x, w, w))
    in_fresh_thread(lambda: kernels.linear_dx(dz, w))
    in_fresh_thread(lambda: kernels.linear_dw(dz, x)[0])


def test_int8_linear_and_attention():
    q, w = (torch.randint(-127, 128, shape, device=DEV, dtype=torch.int8) for shape in ((300, 256), (512, 256)))
    sx, sw = torch.rand(300, device=DEV), torch.rand(512, device=DEV)
    out = torch.empty(300, 512, device=DEV, dtype=torch.bfloat16)

    def gemm():
        kernels.gemm_w8a8_into(q, w, sx, sw, None, out)
        return out.clone()

    in_fresh_thread(gemm)
    x, result = rand(1, 256, 2, 128), rand(1, 256, 2, 128)
    plan = kernels.AttnPlan(1, 2, 256, 256, 128, torch.bfloat16, _lib.MODE_REF)
    plan.prep(x, x)
    in_fresh_thread(lambda: plan.main(x, result, 128 ** -0.5).clone())


def test_first_backward_of_a_process():
    """The autograd engine's thread is new, and the first launch of a projection without bias and
    activation is a product."""
    code = ("import torch; from diffucore_b200 import text\n"
            "x, w = (torch.ones(n, 64, device='cuda', dtype=torch.bfloat16).requires_grad_() for n in (300, 256))\n"
            "y = text.linear(x, w); dy = torch.ones_like(y)\n"
            "dx, dw = torch.autograd.grad(y, (x, w), dy)\n"
            "assert (dx == 256).all() and (dw == 300).all()\n")
    res = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr
