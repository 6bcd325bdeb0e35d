"""Which memory flash_attention_packed takes as `out`: q's, where q is dense, and none that anything else read has, k and v
that are the same tensor as q included (other workgroups read their rows after some have been written)."""
import pytest
import torch

from gpt_triton_amd import kernels


@pytest.fixture
def calls(monkeypatch):
    """The call up to its launch, on CPU tensors."""
    launched = []
    monkeypatch.setattr(kernels, "_on_gpu", lambda *tensors: 0)
    monkeypatch.setattr(kernels, "_call", lambda *args: launched.append(args))
    return launched


def aligned(*shape):
    n = 1
    for s in shape:
        n *= s
    buf = torch.zeros(n + 8, dtype=torch.float16)
    first = -buf.data_ptr() % 16 // 2
    return buf[first:first + n].view(shape)


def test_one_tensor_in_several_places(calls):
    starts = torch.tensor([0, 5])
    x, y, out = aligned(5, 4, 64), aligned(5, 4, 64), aligned(5, 4, 64)
    for args in ((x, x, x), (x, x, y), (x, y, x)):
        with pytest.raises(AssertionError, match="out"):
            kernels.flash_attention_packed(*args, starts, out=x)
        with pytest.raises(AssertionError, match="out"):
            kernels.flash_attention_packed(*args, starts, out=x.view(5, 4, 64))
    assert not calls
    assert kernels.flash_attention_packed(x, x, x, starts, out=out) is out
    assert kernels.flash_attention_packed(x, y, y, starts, out=x) is x
    assert kernels.flash_attention_packed(x, y, y, starts, out=x.view(5, 4, 64)).data_ptr() == x.data_ptr()
    assert kernels.flash_attention_packed(x[:0], x[:0], x[:0], starts, out=x[:0]).shape == (0, 4, 64)
    assert len(calls) == 3


def test_starts_inside_out(calls):
    buf = aligned(8, 4, 64)
    x, y = aligned(7, 4, 64), aligned(7, 4, 64)
    for first, last in ((0, 2), (100, 103), (446, 448)):  # of 7 * 4 * 64 / 4 = 448 int64, the last two of them out's
        starts = buf.view(-1).view(torch.int64)[first:last]
        with pytest.raises(AssertionError, match="out"):
            kernels.flash_attention_packed(x, y, y, starts, out=buf[:7])
    assert not calls
    kernels.flash_attention_packed(x, y, y, buf.view(-1).view(torch.int64)[448:451], out=buf[:7])
    kernels.flash_attention_packed(x, y, y, buf.view(-1).view(torch.int64)[0:3], out=buf[1:])
    assert len(calls) == 2
