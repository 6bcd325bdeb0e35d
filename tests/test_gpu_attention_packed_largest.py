"""Values at the end of fp16's range.  An output is a mean of values, so finite values give a finite one, but its weights
are rounded to fp16 each for the product with v and their sum is not: all rounded up by nearly 2^-11 they make 65536 out of
65504, and what is above 65519 rounds to infinity.

The weights here are 2^6 for the first key and 2^5 (1 + 2^-11 + 2^-16) for the others, which round to 2^5 (1 + 2^-10)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

LARGEST = 65504.0


@pytest.mark.parametrize("heads", [1, 12, 100])
@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
def test_weights_that_all_round_up(gpu_device, d, heads):
    from gpt_triton_amd import kernels as K

    lengths = [600, 1, 1300]
    total = sum(lengths)
    q, k, v = (torch.zeros(total, heads, d, dtype=torch.float16, device=gpu_device) for _ in range(3))
    starts = torch.tensor([0, 600, 601, 1901], device=gpu_device)
    q[..., 0] = 1.0
    k[..., 0] = -1.0
    k[starts[:-1], :, 0] = 0.0
    v[:] = LARGEST
    v[..., 1::2] = -LARGEST
    scale = (1.0 - math.log2(1.0 + 2.0**-11 + 2.0**-16)) * math.log(2.0)
    out = K.flash_attention_packed(q, k, v, starts, scale=scale)
    # half a step of a weight, and of the result
    assert torch.all((out.double() - v.double()).abs() <= LARGEST * (2.0**-11 + 2.0**-11)), out.abs().max()
    # key by key, where a value that is none is among them
    v[600 + 1 + 1299] = math.inf
    out = K.flash_attention_packed(q, k, v, starts, scale=scale)
    assert torch.all((out[:-1].double() - v[:-1].double()).abs() <= LARGEST * (2.0**-11 + 2.0**-11))
    assert torch.all(out[-1] == math.inf)
    v[600 + 1 + 1299] = LARGEST
    v[600 + 1 + 900, :, 0] = -math.inf
    out = K.flash_attention_packed(q, k, v, starts, scale=scale)
    assert torch.all(out[1501:, :, 0] == -math.inf) and torch.all(torch.isfinite(out[:1501]))
