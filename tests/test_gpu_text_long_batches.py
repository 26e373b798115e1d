"""GPU: the embedding's gradient for long batches: right on both sides of each rule on the number of
tokens, and its cost proportional to it."""

from __future__ import annotations

import pytest
import torch

from diffucore_b200 import device_error, kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("T", [95 * 1024, 95 * 1024 + 1, 97 * 1024 + 7, 200_001, (1 << 20) + 5])
@pytest.mark.parametrize("V", [2, 300, 70_000, 600_000])
def test_gradient_of_long_batches(T, V):
    """Small whole numbers: every sum is exact."""
    ids = (torch.rand(T, device=DEV) ** 3 * (V + 1)).long() - 1          # some outside the table: no gradient
    dy = torch.randint(-2, 3, (T, 8), device=DEV)
    got = kernels.embedding_grad(dy.float(), ids, V, padding_idx=1)
    keep = (ids >= 0) & (ids != 1)
    want = torch.zeros(V, 8, device=DEV, dtype=torch.long).index_add_(0, ids[keep], dy[keep])
    assert torch.equal(got.long(), want)
    assert torch.equal(got, kernels.embedding_grad(dy.float(), ids.int(), V, padding_idx=1))
    assert device_error() == 0


def test_cost_is_proportional_to_the_tokens():
    """Eight times the tokens take at most twelve times as long: the sort's counts were once added up with
    the square of the tokens."""
    def microseconds(T):
        ids = (torch.rand(T, device=DEV) ** 3 * 32128).long()
        dy = torch.randn(T, 8, device=DEV)
        for _ in range(3):
            kernels.embedding_grad(dy, ids, 32128)
        best = float("inf")
        for _ in range(5):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            for _ in range(5):
                kernels.embedding_grad(dy, ids, 32128)
            end.record()
            end.synchronize()
            best = min(best, start.elapsed_time(end) * 200)
        return best

    short, long = microseconds(1 << 19), microseconds(1 << 22)
    assert long <= 12 * short, (short, long)
