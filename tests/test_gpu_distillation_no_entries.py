"""Rows for which a teacher has no entries: loss 0 and gradient 0 whatever their logits are."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1, 300, 2049, 20000, 50257, 131072, 200003])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_logits_that_are_no_numbers(gpu_device, dtype, V, bad):
    from gpt_triton_amd import kernels as K

    gen = torch.Generator(device=gpu_device).manual_seed(V)
    wide = torch.randn(6, V + 3, generator=gen, device=gpu_device).to(dtype)
    x = wide[:, 1:V + 1]
    x[1:5, V // 2] = bad
    x[2] = bad
    ids = torch.randint(0, V, (6, 3), generator=gen, device=gpu_device)
    teacher = torch.randn(6, 3, generator=gen, device=gpu_device)
    ids[1:3] = -100  # no token of the vocabulary
    ids[3] = V
    teacher[4] = -math.inf  # no probability
    loss, grad = K.distillation_loss_and_grad(x, ids, teacher, 2.0)
    leaf = x.detach().requires_grad_()
    alone = K.distillation_loss(leaf, ids, teacher, 2.0)
    back, = torch.autograd.grad(alone, leaf, torch.full((6,), 3.0, device=gpu_device))
    for losses, gradient in ((loss, grad), (alone.detach(), back)):
        assert torch.all(losses[1:5] == 0) and torch.all(gradient[1:5] == 0)
        assert torch.all(torch.isfinite(losses)) and torch.all(torch.isfinite(gradient))
    if V > 1:
        assert torch.all((grad[[0, 5]] != 0).any(dim=1))
