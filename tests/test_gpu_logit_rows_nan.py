"""token_log_probs' top tokens in rows that hold NaN, which count as -infinity among them: the ids of the same rows with
-infinity in their place.  A thread has several chunks of 8 (fp16) or 4 logits and perhaps a single one in front of or
behind all chunks, so the largest logits lie in the chunk of a NaN, in another chunk of its thread, and at both ends."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(gpu_device):
    from gpt_triton_amd import kernels

    return kernels


def rows_with_nan(r, V, n):
    """[9, V]: n logits of a 16-byte chunk."""
    x = r.standard_normal((9, V)) * 2.5
    first = int(r.integers(0, V))
    # one NaN beside the largest logit, in its chunk wherever the row begins
    x[0, first], x[0, first - 1 if first else 1] = 20.0, math.nan
    # beside each of the 128 largest, where that is none of them
    top = np.argsort(-x[1])[:min(V, 128)]
    beside = np.setdiff1d((top + 1) % V, top)
    x[1, beside] = math.nan
    # a row's ends
    x[2, [0, V - 1]] = math.nan
    x[2, [1 % V, V // 2, max(V - 2, 0)]] = [19.0, 18.0, 17.0]
    # the chunks of one thread, for every number of threads that a row may have
    for row, threads in ((3, 64), (4, 256), (5, 512), (6, 1024)):
        x[row, V // 3] = 20.0
        x[row, (V // 3 + threads * n) % V] = math.nan
    # every thread has some; and hardly a number is left
    x[7, ::97] = math.nan
    x[8, r.random(V) < 0.97] = math.nan
    return x


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("V", [3, 9, 300, 2047, 5000, 20000, 50257, 65024, 131072, 200003])
def test_nan_beside_the_largest(K, gpu_device, dtype, V):
    r = np.random.default_rng(V)
    n = 16 // torch.finfo(dtype).bits * 8
    x = torch.from_numpy(rows_with_nan(r, V, n)).to(dtype)
    clean = torch.where(torch.isnan(x), -math.inf, x).double().numpy()
    want = np.argsort(-clean, axis=1, kind="stable")
    wide = torch.full((len(x), V + 5), 30.0, dtype=dtype, device=gpu_device)  # rows that begin at every alignment
    wide[:, 3:3 + V] = x
    for view in (x.to(gpu_device), wide[:, 3:3 + V]):
        for top in (1, 5, 20, 32, 40, 64, 128):
            if top <= V:
                s = K.token_log_probs(view, top=top)
                assert np.array_equal(s.top_tokens.cpu().numpy(), want[:, :top]), top
                spoilt = torch.isnan(view).any(dim=1)
                assert torch.equal(torch.isnan(s.top_log_probs).any(dim=1), spoilt)
                assert torch.equal(torch.isnan(s.entropy), spoilt)
