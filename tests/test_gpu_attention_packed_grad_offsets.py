"""Gradients of flash_attention_packed where the keys' and values' channels have offsets, as biases give them.

delta = e . out is subtracted from e . v, whose offsets it has to cancel: u = w (e . v - delta) sums to 0 over a row's keys, so
that offsets of the keys cancel in dq.  With h = 2^-11 the kernels round w and u to fp16 once each, by at most h of themselves,
evenly spread: their squares are h^2 / 3 of the squares.  Roundings of different elements are independent, so
that squares add up, over a query's keys:
  * delta, a mean over weights that the forward pass rounds, is off by sum w^2 (p - delta)^2 h^2 / 3, times (sum w k)^2 in dq
    and (sum w q)^2 over a key's queries in dk; offsets of the values are in all terms of the mean, and play no part;
  * u's rounding: sum u^2 k^2 h^2 / 3, and sum u^2 q^2 h^2 / 3;
  * the result's own: h^2 / 3 of its square.
The 2-norm of all errors is held to 1.5 times the root of the sum.  What fp32 rounds is far below: 2^-24 of sums that
are at most 30 times the spread that h, 2^13 times larger, meets."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

H2 = 2.0**-22 / 3


@pytest.fixture(scope="module")
def K(gpu_device):
    from gpt_triton_amd import kernels

    return kernels


def make(seed, total, n, g, d, offset, device):
    """q, k, v, e of unit spread, channels of k and v with offsets of that size."""
    r = np.random.default_rng(seed)
    new = lambda heads, by: torch.from_numpy(
        (r.standard_normal((total, heads, d)) + by * r.standard_normal((heads, d))).astype(np.float16)).to(device)
    return new(n, 0.0), new(g, offset), new(g, offset), new(n, 0.0)


def want(q, k, v, e, scale):
    """((dq, dk), the expected squares of their errors) of one sequence in 64 bits."""
    L, n, d = q.shape
    rep = n // k.shape[1]
    new = lambda like: torch.zeros(like.shape, dtype=torch.float64, device=q.device)
    dq, dk, sq, sk = new(q), new(k), new(q), new(k)
    past = torch.ones(L, L, dtype=torch.bool, device=q.device).tril_()
    mm = lambda a, b: torch.mm(a, b.contiguous())
    for i in range(n):
        a, b, c, g = q[:, i].double(), k[:, i // rep].double(), v[:, i // rep].double(), e[:, i].double()
        w = torch.softmax(torch.where(past, mm(a, b.t()) * scale, -math.inf), 1)
        p = mm(g, c.t())
        p = p - (w * p).sum(1, keepdim=True)
        u = w * p
        delta = (u * u).sum(1, keepdim=True)
        dq[:, i] = mm(u, b) * scale
        sq[:, i] = (delta * mm(w, b)**2 + mm(u * u, b * b)) * H2 * scale**2
        dk[:, i // rep] += mm(u.t(), a) * scale
        sk[:, i // rep] += (mm((w * w).t(), delta * a * a) + mm((u * u).t(), a * a)) * H2 * scale**2
    return (dq, dk), tuple(s + H2 * x * x for s, x in ((sq, dq), (sk, dk)))


def ratios(K, lengths, n, g, d, offset, device, seed):
    """Errors of dq and dk over what is expected of them, 2-norms, of the rows from the 17th of each text on."""
    q, k, v, e = make(seed, sum(lengths), n, g, d, offset, device)
    starts = torch.tensor([0, *np.cumsum(lengths).tolist()], device=device)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(K.flash_attention_packed(*leaves, starts), leaves, e)
    off, may, at = [0.0, 0.0], [0.0, 0.0], 0
    for L in lengths:
        rows = slice(at, at + L)
        at += L
        exact, squares = want(q[rows], k[rows], v[rows], e[rows], d**-0.5)
        for i in range(2):
            off[i] += float(((got[i][rows].double() - exact[i])**2)[16:].sum())
            may[i] += float(squares[i][16:].sum())
    return [math.sqrt(a / b) for a, b in zip(off, may)]


@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2)])
@pytest.mark.parametrize("offset", [0.0, 1.0, 3.0, 10.0])
def test_offsets(K, gpu_device, d, heads, offset):
    for lengths in ([1024], [40, 300, 129]):
        got = ratios(K, lengths, *heads, d, offset, gpu_device, d + len(lengths))
        assert max(got) <= 1.5, (lengths, got)


@pytest.mark.parametrize("d", [16, 64, 256])
def test_without_the_remainder(K, gpu_device, d):
    """The library's calls that keep none: the same output, gradients within the bounds of a rounded output's delta."""
    from gpt_triton_amd import _lib
    from test_gpu_attention_packed_grad import largest_norm, want as bounds

    lengths, n, g = [40, 300, 129], 4, 2
    T = sum(lengths)
    q, k, v, e = make(d, T, n, g, d, 0.0, gpu_device)
    starts = torch.tensor([0, *np.cumsum(lengths).tolist()], device=gpu_device)
    lib, scale = _lib.load(), d**-0.5
    out, dq, dk, dv = (torch.empty_like(t) for t in (q, q, k, v))
    stats = torch.empty(n, T, 2, device=gpu_device)
    sizes = (len(lengths), T, n, g, d, n * d, d, g * d, d, g * d, d, scale)
    nbytes = lib.gptmi_flash_attn_packed_backward_workspace_bytes(len(lengths), T, n, g, d)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=gpu_device)
    stream, at = torch.cuda.current_stream().cuda_stream, lambda *tensors: [t.data_ptr() for t in tensors]
    assert lib.gptmi_flash_attn_packed_train(*at(q, k, v, out, stats, starts), *sizes, 1, stream) == 0
    assert lib.gptmi_flash_attn_packed_backward(*at(q, k, v, out, stats, e, starts, dq, dk, dv), *sizes, ws.data_ptr(), nbytes,
                                                1, stream) == 0
    assert torch.equal(out, K.flash_attention_packed(q, k, v, starts))
    first = 0
    for L in lengths:
        rows = slice(first, first + L)
        first += L
        for x, y, t in zip((dq, dk, dv), *bounds(q[rows], k[rows], v[rows], e[rows], scale, largest_norm(e) * largest_norm(v))):
            assert torch.all((x[rows].double() - y).abs() <= t)
