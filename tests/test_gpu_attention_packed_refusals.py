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


def test_out_that_overlaps(gpu_device):
    from gpt_triton_amd import kernels as K

    buf = torch.randn(4, 40, 4, 64, device=gpu_device).half()
    q, k, v, out = buf
    starts = torch.tensor([0, 40], device=gpu_device)
    want = K.flash_attention_packed(q, k, v, starts)
    for bad in (k, v, buf.view(-1, 4, 64)[1:41], buf.view(-1, 4, 64)[79:119], buf.view(-1, 4, 64)[81:121]):
        with pytest.raises(AssertionError):
            K.flash_attention_packed(q, k, v, starts, out=bad)
    with pytest.raises(AssertionError):  # q's columns of a product, whose rows are not dense
        wide = torch.randn(40, 12, 64, device=gpu_device).half()
        K.flash_attention_packed(*wide.split(4, dim=1), starts, out=wide.view(-1, 4, 64)[:40])
    assert torch.equal(K.flash_attention_packed(q, k, v, starts, out=out), want)
    assert torch.equal(K.flash_attention_packed(q, k, v, starts, out=q), want)
