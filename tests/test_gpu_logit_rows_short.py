"""Rows of up to 256 chunks of 16 bytes (2048 fp16 or 1024 fp32 logits), which one wavefront sums.

Tolerances (u = 2^-24): a lane has up to 4 chunks and a single logit, at most ceil(V / 64) + 2 terms, of which fp16 ones go to
two sums; 6 additions join the lanes; what a sum is scaled by when its reference moves, in a lane and across, is off by
fewer than 8 u: SUM = u (8 + ceil(V / 64) + 16), where rows of more chunks have at least 256 threads and ceil(V / 256).  A
term e = exp(-t), t = (m - x) / tau, is off by (4 + 3 t) u of itself.  Beside the largest logit's 1, t exp(-t) <= 0.37
leaves 2 u of that in a sum; where the 1 is not part of it, 3 u times the mean of t, weighed by the terms:
  * a log probability is a difference, 3 u t, less a logarithm, SUM and 4 u of itself.  The largest logit's is log(1 + the
    others) alone: SUM + 8 u + 3 u mean t of itself, the others' mean;
  * an entropy is log(1 + the others) and a mean of t, of one sign: 64 u + 2 SUM + 3 u mean t, the mean of terms e t;
  * a gradient's parts are off by 100 u + 2 SUM + 3 u t of their size, t their own logit's, and the result by half a step of what it
    is stored in.  The hardware's exponential is 0 below 2^-126, the least normal number: p as large as that is missing."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24


@pytest.mark.parametrize("V,dtype", [(V, torch.float16) for V in (65, 300, 777, 1023, 1024, 1537, 2047, 2048)] +
                         [(V, torch.float32) for V in (65, 300, 777, 1023, 1024)])
def test_sums_of_a_wavefront(gpu_device, dtype, V):
    from gpt_triton_amd import kernels as K

    r = np.random.default_rng(V)
    rows, tau, error = 37, 0.8, U * (8 + -(-V // 64) + 16)
    # flat, ordinary and sharp rows, and one with all the probability on a token
    x = r.standard_normal((rows, V)) * np.linspace(0.0, 6.0, rows)[:, None]
    x[-1, 5] = 60.0
    wide = torch.zeros(rows, V + 3, dtype=dtype, device=gpu_device)
    wide[:, 2:V + 2] = torch.from_numpy(x)
    leaf = wide[:, 2:V + 2].detach().requires_grad_()
    x = leaf.detach().cpu().double().numpy()
    tokens = r.integers(0, V, rows)
    tokens[-1] = 5
    g, h = (r.standard_normal(rows).astype(np.float32) for _ in range(2))
    ids, teacher = r.integers(0, V, (rows, 6)), r.standard_normal((rows, 6)).astype(np.float32)
    dev = lambda a: torch.from_numpy(a).to(gpu_device)  # noqa: E731
    s = K.token_log_probs(leaf, dev(tokens), top=20, temperature=tau)
    grad, = torch.autograd.grad((s.log_probs, s.entropy), leaf, (dev(g), dev(h)))
    loss, one_pass = K.distillation_loss_and_grad(leaf.detach(), dev(ids), dev(teacher), tau)

    z = x / tau
    z = z - z.max(1, keepdims=True)
    t = -z
    # the sum but for one largest logit's 1, which in 64 bits would swallow the last row's others, of exp(-50)
    first = x.argmax(1)
    others = np.exp(z)
    others[np.arange(rows), first] = 0.0
    z = z - np.log1p(others.sum(1, keepdims=True))
    far = (others * t).sum(1) / others.sum(1)
    farther = (others * t * t).sum(1) / (others * t).sum(1).clip(1e-300)
    p, at = np.exp(z), np.arange(rows)
    host = lambda a: a.detach().cpu().double().numpy()  # noqa: E731
    score = z[at, tokens]
    # of the largest logit, t = 0, a logarithm of a number near 1, which keeps its bits
    tol = 3 * U * t[at, tokens] + np.where(t[at, tokens] == 0, (error + 8 * U + 3 * U * far) * np.abs(score),
                                           error + 4 * U * np.abs(score))
    assert np.all(np.abs(host(s.log_probs) - score) <= tol + 2.0**-149)
    entropy = -(p * z).sum(1)
    assert np.all(np.abs(host(s.entropy) - entropy) <= (64 * U + 2 * error + 3 * U * farther) * entropy + 1e-37)
    order = np.argsort(-x, axis=1, kind="stable")[:, :20]
    assert np.array_equal(host(s.top_tokens), order)
    top = np.take_along_axis(z, order, 1)
    assert np.all(np.abs(host(s.top_log_probs) - top) <= 3 * U * np.take_along_axis(t, order, 1) + error + 4 * U * np.abs(top))

    one = np.zeros_like(p)
    one[at, tokens] = 1.0
    of_p = (np.abs(g)[:, None] + np.abs(h)[:, None] * (np.abs(z) + entropy[:, None])) / tau
    parts = one * np.abs(g)[:, None] / tau + p * of_p
    want = ((one - p) * g[:, None] - h[:, None] * p * (z + entropy[:, None])) / tau
    half = torch.finfo(dtype).eps / 2
    least = 2.0**-25 if dtype == torch.float16 else 2.0**-149
    assert np.all(np.abs(host(grad) - want) <= (100 * U + 2 * error + 3 * U * t) * parts + half * np.abs(want) + least +
                  2.0**-126 * of_p)

    q = np.exp(teacher.astype(np.float64) / tau)
    q /= q.sum(1, keepdims=True)
    there = np.take_along_axis(z, ids, 1)
    size = (q * (np.abs(np.log(q)) + np.abs(there) + 1)).sum(1)
    assert np.all(np.abs(host(loss) - (q * (np.log(q) - there)).sum(1)) <= (U * (32 + 6) + error) * size)
    share = np.zeros_like(p)
    np.add.at(share, (at[:, None], ids), q)
    want = (p - share) / tau
    assert np.all(np.abs(host(one_pass) - want) <= ((100 + 6) * U + 2 * error + 3 * U * t) * (p + share) / tau + half * np.abs(want) +
                  least + 2.0**-126 / tau)
