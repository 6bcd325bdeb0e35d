"""Gradients of flash_attention_packed of texts that lie beside others with far larger gradients or values: what the products'
operands are scaled by goes by a text's own rows, so a text's tolerance has its own largest norms in it, whatever is packed with
it.  A gradient beyond 65504, fp16's largest number, is an infinity of its sign; one that may be, within its tolerance, may."""
import math

import numpy as np
import pytest
import torch

from test_gpu_attention_packed_grad import grads, largest_norm, make, starts_of, want

pytestmark = pytest.mark.gpu

LENGTHS = [300, 40, 129, 0, 700, 1, 77]
# of the output's gradient and of the values, text by text: 10^7 and more between the texts' products
E_SIZES = [1e-3, 1e3, 1e4, 1.0, 2e-3, 1e4, 1.0]
V_SIZES = [1.0, 30.0, 300.0, 1.0, 1e-2, 1.0, 1e-2]


@pytest.fixture(scope="module")
def K(gpu_device):
    from gpt_triton_amd import kernels

    return kernels


def spread(t, sizes, lengths):
    by = torch.tensor(sizes, device=t.device).repeat_interleave(torch.tensor(lengths, device=t.device))
    return (t.float() * by[:, None, None]).half()


def compare(name, x, y, t):
    x = x.double()
    off = (x - y).abs()
    fine = (off <= t) | ((y.abs() + t >= 65504) & (x == math.inf * y.sign()))
    assert torch.all(fine), (name, float((off / t)[~fine].max()))


@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2)])
@pytest.mark.parametrize("many", [False, True])
def test_texts_of_different_sizes(K, gpu_device, d, heads, many):
    """many: among so many more of them that the blocks are dealt in another order."""
    r = np.random.default_rng(d)
    lengths, e_sizes, v_sizes = LENGTHS, E_SIZES, V_SIZES
    if many:
        lengths, e_sizes, v_sizes = lengths + [3] * 300, e_sizes + [1e4] * 300, v_sizes + [100.0] * 300
    q, k, v, e = make(r, sum(lengths), *heads, d, False, gpu_device)
    v, e = spread(v, v_sizes, lengths), spread(e, e_sizes, lengths)
    _, *got = grads(K, q, k, v, e, starts_of(lengths, gpu_device))
    at = 0
    for L in lengths[:len(LENGTHS)]:
        rows = slice(at, at + L)
        at += L
        if L:
            bound = largest_norm(e[rows]) * largest_norm(v[rows])
            for name, x, y, t in zip("qkv", got, *want(q[rows], k[rows], v[rows], e[rows], d**-0.5, bound)):
                compare((name, L), x[rows], y, t)


@pytest.mark.parametrize("d", [64, 256])
def test_long_texts_of_different_sizes(K, gpu_device, d):
    """A largest row far behind in its text, and nothing but zeros in one of them."""
    r = np.random.default_rng(d)
    lengths = [1100, 700, 520]
    q, k, v, e = make(r, sum(lengths), 4, 2, d, False, gpu_device)
    e = spread(e, [1e-3, 1e2, 0.0], lengths)
    e[1090] *= 500.0
    v[1797] *= 100.0
    _, *got = grads(K, q, k, v, e, starts_of(lengths, gpu_device))
    at = 0
    for L in lengths:
        rows = slice(at, at + L)
        at += L
        bound = largest_norm(e[rows]) * largest_norm(v[rows])
        for name, x, y, t in zip("qkv", got, *want(q[rows], k[rows], v[rows], e[rows], d**-0.5, bound)):
            compare((name, L), x[rows], y, t)


@pytest.mark.parametrize("d", [64, 128])
def test_heads_of_different_sizes(K, gpu_device, d):
    """A key head whose queries' gradients are a millionth of another's."""
    r = np.random.default_rng(d)
    L = 400
    q, k, v, e = make(r, L, 4, 2, d, False, gpu_device)
    e = (e.float() * torch.tensor([1e-3, 1e-3, 1e4, 1e4], device=gpu_device)[:, None]).half()
    _, *got = grads(K, q, k, v, e, starts_of([L], gpu_device))
    for g in range(2):
        own = slice(2 * g, 2 * g + 2)
        args = q[:, own], k[:, g:g + 1], v[:, g:g + 1], e[:, own]
        bound = largest_norm(args[3]) * largest_norm(args[2])
        for name, x, y, t in zip("qkv", (got[0][:, own], got[1][:, g:g + 1], got[2][:, g:g + 1]),
                                 *want(*args, d**-0.5, bound)):
            compare((name, g), x, y, t)
