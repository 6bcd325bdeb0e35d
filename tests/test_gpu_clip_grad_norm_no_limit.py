"""clip_grad_norm_ without a limit, of gradients that are no numbers: what is written says that the step is one to skip, and
the norm says so in any case."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16


@pytest.fixture(scope="module")
def K(gpu_device):
    from gpt_triton_amd import kernels

    return kernels


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("scale", [1.0, 0.5])
@pytest.mark.parametrize("to", [None, F32, F16, "some"])
def test_no_numbers(K, gpu_device, dtype, bad, scale, to):
    r = torch.Generator().manual_seed(0)
    grads = [torch.randn(n, generator=r).to(gpu_device, dtype) for n in (5000, 72_778, 3)]
    grads[1][4000] = bad
    kept = [g.clone() for g in grads]
    if to is None:
        out = None
    elif to == "some":
        out = [grads[0], torch.zeros_like(grads[1]), grads[2]]
    else:
        out = [torch.zeros_like(g, dtype=to) for g in grads]
    norm = float(K.clip_grad_norm_(grads, math.inf, scale=scale, out=out))
    assert math.isnan(norm) if math.isnan(bad) else norm == math.inf
    if out is None and scale == 1.0:  # the norm alone
        assert all(torch.equal(g.nan_to_num(), k.nan_to_num()) for g, k in zip(grads, kept))
        return
    for o in grads if out is None else out:
        assert torch.all(torch.isnan(o) | (o == 0))


@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_numbers(K, gpu_device, scale):
    g = torch.randn(9000, device=gpu_device)
    kept, out = g.clone(), torch.empty_like(g)
    K.clip_grad_norm_([g], math.inf, scale=scale, out=[out])
    assert torch.equal(out, kept * scale) and torch.equal(g, kept)
    K.clip_grad_norm_([g], math.inf, scale=scale)
    assert torch.equal(g, out)
