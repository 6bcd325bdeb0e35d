"""Gradients of packed attention and of the embeddings under torch's checkpoints, which form the forward pass again and let what
it saves be read once."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(gpu_device):
    from gpt_triton_amd import kernels

    return kernels


@pytest.mark.parametrize("reentrant", [False, True])
def test_attention(K, gpu_device, reentrant):
    q, k, v, e = (torch.randn(70, n, 64, device=gpu_device).half() for n in (4, 2, 2, 4))
    starts = torch.tensor([0, 30, 70], device=gpu_device)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    call = lambda *t: K.flash_attention_packed(*t, starts)
    want = torch.autograd.grad(call(*leaves), leaves, e)
    checkpoint(call, *leaves, use_reentrant=reentrant).backward(e)
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))


@pytest.mark.parametrize("reentrant", [False, True])
def test_embeddings(K, gpu_device, reentrant):
    ids = torch.randint(0, 50, (3, 20), device=gpu_device)
    tables = [torch.randn(n, 64, device=gpu_device).requires_grad_() for n in (50, 32)]
    e = torch.randn(3, 20, 64, device=gpu_device)
    call = lambda *t: K.fused_embeddings(ids, *t)
    want = torch.autograd.grad(call(*tables), tables, e)
    checkpoint(call, *tables, use_reentrant=reentrant).backward(e)
    assert all(torch.equal(t.grad, w) for t, w in zip(tables, want))
