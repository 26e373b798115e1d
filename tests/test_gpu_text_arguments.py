"""GPU: the single steps of the text operators (diffucore_b200.kernels) refuse tensors that do not
belong together before anything is launched, and take any layout of those that do; tensors whose
memory does not hold their values as they are (negated views, zero tensors without memory)."""

from __future__ import annotations

import pytest
import torch

from diffucore_b200 import _lib, device_error, kernels, text

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device=DEV).to(dtype)


def refuses(error, why, call, *args, **kw):
    with pytest.raises(error, match=why):
        call(*args, **kw)


def test_products_of_the_backward_pass_refuse():
    dz, w, x = rand(20, 32), rand(32, 48), rand(20, 48)
    dx, dw = kernels.linear_dx, kernels.linear_dw
    refuses(ValueError, "does not match w", dx, dz, rand(31, 48))
    refuses(ValueError, "does not match w", dx, dz, rand(33, 48))
    refuses(ValueError, "matrices", dx, dz[0], w)
    refuses(ValueError, "matrices", dx, dz, w[0])
    refuses(TypeError, "w is", dx, dz, w.half())
    refuses(TypeError, "w is", dx, dz, w.cpu())
    refuses(TypeError, "dtype", dx, dz.float(), w.float())
    refuses(RuntimeError, "CUDA tensors only", dx, dz.cpu(), w.cpu())
    refuses(ValueError, "go together", dx, dz, w, dz)
    refuses(ValueError, "go together", dx, dz, w, None, w)
    refuses(ValueError, "dz1", dx, dz, w, rand(19, 32), w)
    refuses(ValueError, "w1", dx, dz, w, dz, rand(32, 47))
    refuses(TypeError, "dz1 is", dx, dz, w, dz.cpu(), w)
    refuses(TypeError, "w1 is", dx, dz, w, dz, w.cpu())
    refuses(ValueError, "does not match x", dw, dz, rand(19, 48))
    refuses(ValueError, "does not match x", dw, dz, rand(21, 48))
    refuses(ValueError, "matrices", dw, dz, x[0])
    refuses(TypeError, "x is", dw, dz, x.half())
    refuses(TypeError, "x is", dw, dz, x.cpu())
    refuses(ValueError, "dz1", dw, dz, x, rand(20, 31))
    refuses(TypeError, "dz1 is", dw, dz, x, dz.half())


def test_pointwise_gradient_refuses():
    dy, z = rand(20, 30), torch.randn(20, 32, device=DEV)
    call = kernels.act_grad
    refuses(TypeError, "dtype", call, dy.float(), z, None, "silu")
    refuses(RuntimeError, "CUDA tensors only", call, dy.cpu(), None, None, None, True)
    refuses(ValueError, "dy must be", call, dy[0], None, None, None, True)
    refuses(TypeError, "z is", call, dy, z.to(torch.bfloat16), None, "silu")
    refuses(TypeError, "z is", call, dy, z.cpu(), None, "silu")
    refuses(ValueError, "kept pre-activation", call, dy, z[:19], None, "silu")
    refuses(ValueError, "kept pre-activation", call, dy, z[:, :29], None, "silu")
    refuses(ValueError, "kept pre-activation", call, dy, z[0], None, "silu")
    refuses(ValueError, "kept pre-activation", call, dy, torch.randn(32, 20, device=DEV).t(), None, "silu")
    refuses(ValueError, "must hold 32", call, dy, torch.randn(20, 30, device=DEV), None, "silu")
    refuses(ValueError, "goes with z", call, dy, None, z, "silu")
    refuses(ValueError, "kept pre-activation", call, dy, z, z[:19], "silu")
    refuses(ValueError, "row stride", call, dy, z, torch.randn(20, 36, device=DEV), "silu")
    refuses(ValueError, "needs z1", call, dy, z, None, "silu", False, True)
    refuses(RuntimeError, "no rows", call, dy[:0], z[:0], None, "silu")


def test_norm_gradient_refuses():
    x, dy, w = rand(20, 32), rand(20, 32), rand(32)
    _, mean, rstd = kernels.layer_norm(x, w, None, 1e-5, keep_stats=True)
    call = kernels.layer_norm_grad
    refuses(ValueError, "does not match x", call, dy[:19], x, w, mean, rstd)
    refuses(ValueError, "does not match x", call, rand(20, 31), x, w, mean, rstd)
    refuses(ValueError, "does not match x", call, dy[0], x[0], w, mean, rstd)
    refuses(TypeError, "x is", call, dy, x.half(), w, mean, rstd)
    refuses(TypeError, "x is", call, dy, x.cpu(), w, mean, rstd)
    refuses(ValueError, "weight", call, dy, x, w[:31], mean, rstd)
    refuses(TypeError, "weight", call, dy, x, w.half(), mean, rstd)
    refuses(TypeError, "weight", call, dy, x, w.cpu(), mean, rstd)
    refuses(ValueError, "mean", call, dy, x, w, mean[:19], rstd)
    refuses(ValueError, "rstd", call, dy, x, w, mean, rstd[:, None])
    refuses(TypeError, "mean", call, dy, x, w, mean.half(), rstd)
    refuses(TypeError, "rstd", call, dy, x, w, mean, rstd.cpu())
    refuses(TypeError, "gradients in", call, dy, x, w, mean, rstd, dtype=torch.float16)
    refuses(ValueError, "x must be", kernels.layer_norm, x[0], None, None, 1e-5)
    refuses(ValueError, "x must be", kernels.layer_norm, x[None], None, None, 1e-5)


def test_lookup_steps_refuse():
    ids = torch.zeros(6, dtype=torch.long, device=DEV)
    refuses(ValueError, "table must be", kernels.embedding, ids, rand(4, 8, 2))
    refuses(ValueError, "table must be", kernels.embedding, ids, rand(8))
    refuses(ValueError, "dy must be", kernels.embedding_grad, rand(6, 8, 2), ids, 4)
    refuses(ValueError, "dy must be", kernels.embedding_grad, rand(6), ids, 4)
    refuses(RuntimeError, "bad shape", kernels.embedding_grad, rand(6, 8), ids, 0)
    refuses(ValueError, "matrix", kernels.matrix_operand, rand(8))


def test_second_operands_of_another_layout():
    """dz1 and w1 (dw: dz1) in rows of another pitch than dz's, or unaligned: small whole numbers, so that
    every product and sum is exact."""
    def whole(*shape):
        return torch.randint(-3, 4, shape, device=DEV).to(torch.bfloat16)

    def layouts(t):
        wide = torch.zeros(t.shape[0], t.shape[1] + 24, device=DEV, dtype=t.dtype)
        for at in (0, 8, 3):
            view = wide[:, at:at + t.shape[1]]
            view.copy_(t)
            yield view.clone(memory_format=torch.preserve_format) if at == 8 else view
        yield t.t().contiguous().t()

    for N in (32, 31):
        dz, dz1, w, w1, x = whole(20, N), whole(20, N), whole(N, 40), whole(N, 40), whole(20, 40)
        want = (dz.double() @ w.double() + dz1.double() @ w1.double()).to(torch.bfloat16)
        wants = [(d.double().t() @ x.double()).to(torch.bfloat16) for d in (dz, dz1)]
        for a in layouts(dz):
            for b in layouts(dz1):
                for c in layouts(w1):
                    assert torch.equal(kernels.linear_dx(a, w, b, c), want)
                got = kernels.linear_dw(a, x, b)
                assert all(torch.equal(p, q) for p, q in zip(got, wants))


@pytest.mark.parametrize("N", [32, 30, 1])
def test_pointwise_gradient_of_kept_values(N):
    """The kept pre-activations as the forward calls return them, whole or narrowed to N columns."""
    x, w, dy = rand(20, 16), rand(N, 16), rand(20, N)
    _, z = kernels.linear(x, w, act="relu", keep_z=True)
    want = torch.where(z[:, :N] > 0, dy, torch.zeros_like(dy))
    for kept in (z, z[:, :N]):
        dz, _, db, _ = kernels.act_grad(dy, kept, None, "relu", True)
        assert torch.equal(dz, want)
        assert db.shape == (N,)


def test_norm_gradient_keeps_an_fp32_weight():
    """Gradients asked for in 16 bits are rounded at the end; the fp32 weight is not."""
    x, dy, w = rand(300, 64), rand(300, 64), torch.rand(64, device=DEV) + 0.5
    _, mean, rstd = kernels.layer_norm(x, w, None, 1e-5, keep_stats=True)
    want = kernels.layer_norm_grad(dy, x, w, mean, rstd)
    got = kernels.layer_norm_grad(dy, x, w, mean, rstd, dtype=torch.bfloat16)
    assert torch.equal(got[0], want[0])
    assert all(g.dtype == torch.bfloat16 and torch.equal(g, e.to(torch.bfloat16)) for g, e in zip(got[1:], want[1:]))


def test_negated_views():
    """torch._neg_view(t) has t's memory and -t's values, as the imaginary part of a conjugate has."""
    x, w, b, r = rand(40, 48), rand(56, 48), rand(56), rand(40, 56)
    neg = torch._neg_view

    def same(call, *args):
        def step(leaves, dy):
            y = call(*leaves)
            return (call(*[a.detach() for a in leaves]), y.detach(), *torch.autograd.grad(y, leaves, dy))

        ones = torch.ones_like(call(*args))
        want = step([a.neg().requires_grad_() for a in args], -ones)
        got = step([neg(a).requires_grad_() for a in args], neg(ones))
        for p, q in zip(want, got):
            assert torch.equal(p, q) and not q.is_neg()

    same(lambda x, w, b, r: text.linear(x, w, b, activation="silu", residual=r), x, w, b, r)
    same(lambda x, w, b, r: text.linear(x[:4, 1:], w[:, 1:], b, residual=r[:4]), x, w, b, r)
    same(text.gated_linear, x, w, rand(56, 48), b, rand(56))
    same(text.layer_norm, x, rand(48), rand(48))
    ids = torch.randint(0, 40, (300,), device=DEV)
    same(lambda t: text.embedding(ids, t), x)
    z = torch.randn(7, 32, device=DEV, dtype=torch.complex64)
    assert z.conj().imag.is_neg()
    assert torch.equal(text.layer_norm(z.conj().imag), text.layer_norm(-z.imag))


def test_zero_tensors_without_memory():
    zero = torch._efficientzerotensor((40, 48), device=DEV, dtype=torch.bfloat16)
    w = rand(56, 48)
    assert not text.linear(zero, w).any() and not text.gated_linear(zero, w, w).any()
    assert not text.layer_norm(zero).any()
    x = rand(40, 48).requires_grad_()
    dx, = torch.autograd.grad(text.layer_norm(x), x, zero)
    assert not dx.any()


def test_both_error_words_are_reported():
    """A wait that timed out and a token id outside its table, both before the words are read: each is
    returned once."""
    while device_error():
        pass
    text.embedding(torch.tensor([10], device=DEV), rand(10, 32))
    status = torch.zeros(1, device=DEV, dtype=torch.int32)
    lib = _lib.load()
    _lib.check(lib.dc_selftest_wait_timeout(2_000_000, status.data_ptr(), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert device_error(clear=False) == 2
    assert device_error() == 2
    assert device_error() == 3
    assert device_error() == 0
    text.embedding(torch.tensor([10], device=DEV), rand(10, 32))
    lib.dc_device_error(None, 1)                             # clears both
    assert device_error() == 0
