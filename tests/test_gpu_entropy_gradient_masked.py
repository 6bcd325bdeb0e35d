"""The entropy's gradient in rows with tokens that cannot occur (logits of -infinity), for gradients of the entropy as large as
fp32 has: 0 for those tokens, and for the others what the formula gives, dH/dx_j = -h p_j (log p_j + H).

Tolerance: with h a power of two the gradient is h times that of h = 1, whose parts p |log p| and p H are off by (100 + 2 (8
+ ceil(V / 64) + 16)) 2^-24 (a term of p by 4 + 3 |log p| roundings, the sums by their additions, at most ceil(V / 64) + 16
a thread and across threads)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("V", [9, 300, 2049, 50257, 200003])
@pytest.mark.parametrize("h", [1.0, 2.0**28, 2.0**30, 2.0**60, 2.0**100])
def test_masked_tokens(gpu_device, dtype, V, h):
    from gpt_triton_amd import kernels as K

    r = np.random.default_rng(V)
    x = torch.from_numpy(r.standard_normal((3, V)) * 2.5).to(dtype)
    hidden = torch.from_numpy(r.random((3, V)) < 0.5)
    hidden[:, V // 2] = False
    x[hidden] = -math.inf
    leaf = x.to(gpu_device).requires_grad_()
    s = K.token_log_probs(leaf)
    grad, = torch.autograd.grad(s.entropy, leaf, torch.full((3,), h, device=gpu_device))
    grad = grad.cpu().double()
    assert torch.all(grad[hidden] == 0)
    z = torch.log_softmax(x.double(), 1)
    p = z.exp()
    terms = torch.where(hidden, 0.0, p * z)
    entropy = -terms.sum(1, keepdim=True)
    want = -h * (terms + p * entropy)
    tol = (100 + 2 * (8 + -(-V // 64) + 16)) * U * h * (terms.abs() + p * entropy)
    if dtype == torch.float16:
        tol = tol + want.abs() * 2.0**-11 + 2.0**-25
        fits = want.abs() <= 65000
        assert torch.all((grad - want).abs()[fits] <= tol[fits])
    else:
        assert torch.all((grad - want).abs() <= tol + 2.0**-149)
