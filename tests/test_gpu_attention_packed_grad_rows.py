"""flash_attention_packed of rows longer than its gradients read: the output all the same, an error in the backward pass."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(gpu_device):
    from gpt_triton_amd import kernels

    return kernels


@pytest.mark.parametrize("T", [1, 3])
def test_long_rows(K, gpu_device, T):
    """Heads one behind the other, as far as a row of q may be pitched."""
    n, d = (1 << 18) + 2, 64
    q = torch.randn(n, T, d, device=gpu_device).half().transpose(0, 1)
    k, v = (torch.randn(T, 2, d, device=gpu_device).half() for _ in range(2))
    starts = torch.tensor([0, T], device=gpu_device)
    want = K.flash_attention_packed(q, k, v, starts)
    q.requires_grad_()
    out = K.flash_attention_packed(q, k, v, starts)
    assert torch.equal(out, want) and out.requires_grad
    with pytest.raises(NotImplementedError, match="no gradient"):
        out.backward(torch.ones_like(out))
    assert q.grad is None
