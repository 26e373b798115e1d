"""The prompt adapter on a GPU: forward and every parameter's gradient against a float64 restatement, a
short training run, and its context through a small FLUX DiT."""

from __future__ import annotations

import math

import pytest
import torch

from diffucore_b200 import _lib, prompt

pytestmark = pytest.mark.gpu
DEV = "cuda"


def restated(adapter: prompt.PromptAdapter, p: dict, ids: torch.Tensor) -> torch.Tensor:
    def norm(x, name):
        c = x - x.mean(-1, keepdim=True)
        return c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * p[name + ".weight"] + p[name + ".bias"]

    x = p["embed.weight"][ids] * adapter.embed.scale
    for i in range(len(adapter.blocks)):
        b = f"blocks.{i}."
        h = norm(x, b + "norm")
        g = h @ p[b + "ff.gate.weight"].t()
        x = x + (g * torch.sigmoid(g) * (h @ p[b + "ff.up.weight"].t())) @ p[b + "ff.down.weight"].t()
    return norm(x, "norm") @ p["proj.weight"].t() + p["proj.bias"]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_adapter_matches_float64(dtype):
    torch.manual_seed(3)
    a = prompt.PromptAdapter(500, 96, 200, 72, depth=2, padding_idx=0, device=DEV, dtype=dtype)
    with torch.no_grad():
        for q in a.parameters():                        # biases and norms away from their initial values
            if q.dim() == 1:
                q.add_(torch.randn_like(q) * 0.1)
    ids = torch.randint(0, 500, (3, 41), device=DEV)
    dy = torch.randn(3, 41, 72, device=DEV).to(dtype)
    params = dict(a.named_parameters())
    out = a(ids)
    got = dict(zip(params, torch.autograd.grad(out, list(params.values()), dy)))
    d = {n: t.detach().double().requires_grad_() for n, t in params.items()}
    want_out = restated(a, d, ids)
    want = dict(zip(d, torch.autograd.grad(want_out, list(d.values()), dy.double())))
    want["embed.weight"][0] = 0                         # the padding token
    # Every value that passes from one operator to the next is rounded to the type: forward 3 per
    # block (norm, product, residual sum) and 3 more (embedding, norm, output), backward as many
    # again plus the dz of each projection. Independent roundings of unit u (2^-9 or 2^-12 relative)
    # add up in squares; 12 forward and 30 in a gradient bound them, times 3 for the amplification
    # of a norm's and an activation's slope.
    u = 2.0 ** (-9 if dtype == torch.bfloat16 else -12)

    def rel(x, y):
        return ((x.double() - y).norm() / y.norm()).item()

    assert rel(out.detach(), want_out.detach()) < 3 * math.sqrt(12) * u
    for n in params:
        assert rel(got[n], want[n]) < 3 * math.sqrt(30) * u, n


def test_training_lowers_the_loss_and_repeats():
    def run():
        torch.manual_seed(1)
        a = prompt.PromptAdapter(300, 128, 256, 64, depth=1, padding_idx=0, device=DEV)
        ids = torch.randint(0, 300, (4, 20), device=DEV)
        target = torch.randn(4, 20, 64, device=DEV).to(torch.bfloat16)
        pad = a.embed.weight[0].clone()
        losses = prompt.fit_context(a, ids, target, 30, lr=2e-3)
        assert torch.equal(a.embed.weight[0], pad)
        return losses

    first = run()
    assert first[-1] < 0.5 * first[0]
    assert run() == first                               # every sum has a fixed order


def test_command_runs_through_the_dit(capsys):
    prompt.main(["--steps", "5", "--prompts", "2", "--tokens", "24", "--vocab", "600", "--dim", "128", "--hidden", "192",
                 "--context", "64", "--depth", "1"])
    said = capsys.readouterr().out
    assert "finite True" in said and "loss" in said
    assert _lib.device_error() == 0
