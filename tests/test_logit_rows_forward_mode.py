"""Scores and losses have no forward-mode derivative: a tensor with a tangent is refused, in front of everything else, and no
tangent is lost without a word."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from gpt_triton_amd import kernels


@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(requires_grad):
    x = torch.randn(2, 8).requires_grad_(requires_grad)
    t = torch.zeros(2, dtype=torch.int64)
    ids, teacher, weights = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3), torch.ones(2)
    with forward_ad.dual_level():
        def dual(a):
            return forward_ad.make_dual(a, torch.ones_like(a))

        calls = [lambda: kernels.token_log_probs(dual(x), t), lambda: kernels.token_log_probs(dual(x), top=2)]
        for loss in (kernels.distillation_loss, kernels.distillation_loss_and_grad):
            calls += [lambda loss=loss: loss(dual(x), ids, teacher), lambda loss=loss: loss(x, ids, dual(teacher)),
                      lambda loss=loss: loss(x, ids, teacher, 1.0, dual(weights))]
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        # without a tangent they go on, to the next refusal
        for call in (lambda: kernels.token_log_probs(x, t), lambda: kernels.distillation_loss(x, ids, teacher, 1.0, weights)):
            with pytest.raises(RuntimeError, match="GPU"):
                call()
