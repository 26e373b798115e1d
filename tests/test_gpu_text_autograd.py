"""GPU: what the text operators do about derivatives they do not have: they are refused, not left out of
a result without a word."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from diffucore_b200 import kernels, text

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device=DEV).to(dtype)


def calls():
    """(name, arguments, function of the arguments) of every differentiable function."""
    ids = torch.randint(0, 9, (6,), device=DEV)
    return [
        ("linear", [rand(6, 16), rand(8, 16), rand(8), rand(6, 8)],
         lambda x, w, b, r: text.linear(x, w, b, activation="silu", residual=r)),
        ("odd linear", [rand(6, 15), rand(7, 15), rand(7), rand(6, 7)],
         lambda x, w, b, r: text.linear(x, w, b, residual=r)),
        ("gated_linear", [rand(6, 16), rand(8, 16), rand(8, 16), rand(8), rand(8)], text.gated_linear),
        ("layer_norm", [rand(6, 16), rand(16), rand(16)], text.layer_norm),
        ("embedding", [rand(9, 16)], lambda table: text.embedding(ids, table)),
    ]


@pytest.mark.parametrize("reverse", [False, True])
def test_forward_mode_tangents_are_refused(reverse):
    for name, args, call in calls():
        for i in range(len(args)):
            with fwd.dual_level():
                given = [a.clone().requires_grad_(reverse) for a in args]
                given[i] = fwd.make_dual(given[i], torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*given)
        call(*args)                                         # the same call without a tangent


def test_forward_mode_tangent_of_the_incoming_gradient_is_refused():
    for name, args, call in calls():
        leaves = [a.clone().requires_grad_() for a in args]
        y = call(*leaves)
        with fwd.dual_level():
            dy = fwd.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaves[:1], dy)


def test_forward_mode_tangents_are_refused_by_single_steps():
    x, w = rand(6, 16), rand(8, 16)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: kernels.linear(dual, w), lambda: kernels.gated_linear(dual, w, w),
                     lambda: kernels.layer_norm(dual, None, None, 1e-5), lambda: kernels.linear_dx(dual, rand(16, 8)),
                     lambda: kernels.linear_dw(rand(6, 8), dual), lambda: kernels.act_grad(dual, None, None, None, True)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


@pytest.mark.parametrize("transform", [torch.func.vmap, torch.func.grad, "jvp"])
def test_function_transforms_are_refused(transform):
    x, w = rand(6, 16), rand(8, 16)
    for call in (lambda t: text.linear(t, w), lambda t: text.layer_norm(t), lambda t: text.gated_linear(t, w, w)):
        with pytest.raises(RuntimeError):
            if transform == "jvp":
                torch.func.jvp(call, (x,), (x,))
            elif transform is torch.func.grad:
                transform(lambda t: call(t).sum())(x)
            else:
                transform(call)(x)


def test_second_derivative_is_refused_where_the_loss_reaches_the_input_by_another_way_too():
    """loss = sum(dx^2) + sum(x^2): without the first term's derivative the gradient would be 2 x."""
    for name, args, call in calls():
        for i in range(len(args)):
            leaves = [a.clone().requires_grad_() for a in args]
            y = call(*leaves)
            first = torch.autograd.grad(y.float().square().sum(), leaves, create_graph=True)
            for g in first:
                with pytest.raises(RuntimeError, match="differentiated twice"):
                    torch.autograd.grad(g.float().square().sum() + leaves[i].float().square().sum(), leaves[i],
                                        retain_graph=True)
            # what does not pass through a gradient is differentiated as ever
            plain, = torch.autograd.grad(leaves[i].float().square().sum(), leaves[i])
            assert torch.equal(plain, (2 * leaves[i].detach().float()).to(plain.dtype))


def test_second_derivative_is_refused_through_the_incoming_gradient():
    for name, args, call in calls():
        leaves = [a.clone().requires_grad_() for a in args]
        y = call(*leaves)
        dy = torch.ones_like(y).requires_grad_()
        g, *_ = torch.autograd.grad(y, leaves, dy, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated twice"):
            torch.autograd.grad(g.float().sum() + dy.float().sum(), dy)
