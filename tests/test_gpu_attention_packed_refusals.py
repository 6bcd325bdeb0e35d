"""What flash_attention_packed refuses of tensors on the GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_refusals(gpu_device):
    from gpt_triton_amd import kernels

    y = torch.zeros(8, 8, 64, dtype=torch.float16, device=gpu_device)
    q, k, v = y.split((4, 2, 2), dim=1)
    starts = torch.tensor([0, 3, 8], device=gpu_device)
    call = kernels.flash_attention_packed
    wide = torch.zeros(8, 2, 72, dtype=torch.float16, device=gpu_device)
    odd = torch.zeros(8, 2, 68, dtype=torch.float16, device=gpu_device)
    for args, more, error in (((q, k, v, starts.cpu()), {}, RuntimeError), ((q, k, v, starts), dict(scale=0.0), ValueError),
                              ((q, k, v, starts), dict(scale=float("nan")), ValueError),
                              ((q, k, v, starts), dict(out=q), AssertionError),
                              ((q, k, v, starts), dict(out=torch.zeros(8, 4, 64, device=gpu_device)), AssertionError),
                              ((q, k, wide[:, :, 4:68], starts), {}, NotImplementedError),
                              ((q, odd[:, :, :64], v, starts), {}, NotImplementedError),
                              ((q, k.transpose(1, 2).contiguous().transpose(1, 2), v, starts), {}, AssertionError)):
        with pytest.raises(error):
            call(*args, **more)
    empty = call(q[:0], k[:0], v[:0], torch.tensor([0, 0], device=gpu_device))
    assert empty.shape == (0, 4, 64)
