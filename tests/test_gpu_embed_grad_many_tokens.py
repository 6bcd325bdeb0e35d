"""Gradients of fused_embeddings over so many tokens that launches of their own add the tiles' counts.  Whole numbers: the sums are
exact in fp32, and compared bit by bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(gpu_device):
    from gpt_triton_amd import kernels

    return kernels


def step(K, ids, dz, V, P):
    wte, wpe = (torch.zeros(n, dz.shape[2], device=dz.device).requires_grad_() for n in (V, P))
    return torch.autograd.grad(K.fused_embeddings(ids, wte, wpe), (wte, wpe), dz)


# 4096 tokens a tile: 400 tiles, one more with a single token, 751 and 1024 in groups of 256
@pytest.mark.parametrize("B,L", [(1600, 1024), (1638401, 1), (3073, 1000), (1025, 4091)])
@pytest.mark.parametrize("V,H", [(50257, 4), (7, 3), (513, 8), (300000, 1)])
def test_many_tokens(K, gpu_device, B, L, V, H):
    r = torch.Generator().manual_seed(B)
    ids = (torch.rand(B, L, generator=r)**3 * (V + 1)).long().to(gpu_device)  # some of them the unknown V
    ids[0, 0], ids[-1, -1] = V - 1, 0
    dz = torch.randint(-2, 3, (B, L, H), generator=r).float().to(gpu_device)
    d_wte, d_wpe = step(K, ids, dz, V, L + 2)
    flat, known = ids.view(-1), ids.view(-1) < V
    want = torch.zeros(V, H, dtype=torch.float64, device=gpu_device)
    want.index_add_(0, flat[known], dz.view(-1, H)[known].double())
    assert torch.equal(d_wte.double(), want)
    assert torch.equal(d_wpe[:L].double(), dz.double().sum(0)) and not d_wpe[L:].any()


def test_same_bits(K, gpu_device):
    """And in the order of the positions: a sum that rounds at each step has the bits of every other call's."""
    r = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 1000, (2000, 1024), generator=r).to(gpu_device)
    dz = torch.randn(2000, 1024, 4, generator=r).to(gpu_device)
    first = step(K, ids, dz, 1000, 1024)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(first, step(K, ids, dz, 1000, 1024)))
