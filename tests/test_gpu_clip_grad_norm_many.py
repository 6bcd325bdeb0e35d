"""clip_grad_norm_ of more tensors than a few launches take, whose workgroups' sums are added in a launch of their own."""
import math

import pytest
import torch

from test_gpu_clip_grad_norm import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(gpu_device):
    from gpt_triton_amd import kernels

    return kernels


def make(count, size, dtype, device, seed=0):
    flat = torch.randn(count * size, generator=torch.Generator().manual_seed(seed)).to(device, dtype)
    return list(flat.split(size))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("max_norm", [0.5, 1e9, math.inf])
@pytest.mark.parametrize("count,size", [(2048, 13), (2049, 13), (2500, 40), (7000, 3), (320, 90_000)])
def test_many(K, gpu_device, dtype, max_norm, count, size):
    first = check(K, make(count, size, dtype, gpu_device), max_norm)
    assert torch.equal(first, check(K, make(count, size, dtype, gpu_device), max_norm))
    out = [torch.empty(size, device=gpu_device) for _ in range(count)] if count < 3000 else None
    check(K, make(count, size, dtype, gpu_device), max_norm, 0.25, out)


def test_captured(K, gpu_device):
    grads = make(2500, 40, torch.float32, gpu_device)
    out = [torch.empty_like(g) for g in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.clip_grad_norm_(grads, 1.0, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = K.clip_grad_norm_(grads, 1.0, out=out)
    for n in range(3):
        for g, x in zip(grads, make(2500, 40, torch.float32, gpu_device, n)):
            g.copy_(x * 10.0**n)
        graph.replay()
        torch.cuda.synchronize()
        eager = [torch.empty_like(o) for o in out]
        assert torch.equal(norm, K.clip_grad_norm_(grads, 1.0, out=eager))
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_too_many(K, gpu_device):
    empty = torch.empty(0, device=gpu_device)
    assert float(K.clip_grad_norm_([empty] * 2**20, 1.0)) == 0.0
    with pytest.raises(NotImplementedError, match="beyond the supported"):
        K.clip_grad_norm_([empty] * (2**20 + 1), 1.0)
