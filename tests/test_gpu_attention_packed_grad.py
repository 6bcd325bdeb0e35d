"""Gradients of flash_attention_packed against their formulas in 64 bits.

With e the output's gradient, p = e . v, delta = e . out, x = w (p - delta), u = 2^-24 (half a step of fp32), h = 2^-11 (of
fp16) the kernels' errors are at most
  * E, of a weight relative to itself: a score is off by (d + 8) u times the sum of its terms' sizes times the scale, its
    exponent and the row's logarithm are rounded at the same size (8 u of it), the denominator by (L + 16) u;
  * w as an operand: h w, at least the step of 2^14 w among subnormal numbers, 2^-39;
  * p: (d + 8) u sum |e| |v|;   delta: (d + 8) u sum |e| |out| and sum |e| times what the output is off by, which is
    (h + 2 E + (L + 8) u) sum w |v| + L 2^-25 max |v| + h |out| + 2^-25;
  * x: w (E |p - delta| + those of p and delta) and, as an operand, h |x|, at least 2^-39 / f where f times B = the product of
    the largest norms of rows of e and v is more than 3.99: 2^-40 B;
  * sums of n terms in fp32: (n + 8) u of the sum of their sizes; the results: h of themselves, at least 2^-25.
The tolerance is their sum, through the products with |k|, |q| and |e|."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U, H, S = 2.0**-24, 2.0**-11, 2.0**-25


@pytest.fixture(scope="module")
def K(gpu_device):
    from gpt_triton_amd import kernels

    return kernels


def largest_norm(t):
    n = t.double().pow(2).sum(-1)
    n = n[torch.isfinite(n)]
    return float(n.max().sqrt()) if n.numel() else 0.0


def want(q, k, v, e, scale, bound, summed=0):
    """((dq, dk, dv), their tolerances) of one sequence in 64 bits.  summed: so many of the first queries' deltas are sums over
    their keys, off by what their terms are and (summed + 16) u of the sizes'."""
    L, n, d = q.shape
    rep = n // k.shape[1]
    new = lambda like: torch.zeros(like.shape, dtype=torch.float64, device=q.device)
    dq, dk, dv, tq, tk, tv = new(q), new(k), new(k), new(q), new(k), new(k)
    past = torch.ones(L, L, dtype=torch.bool, device=q.device).tril_()
    mm = lambda a, b: torch.mm(a, b.contiguous())
    for i in range(n):
        a, b, c, g = q[:, i].double(), k[:, i // rep].double(), v[:, i // rep].double(), e[:, i].double()
        w = torch.softmax(torch.where(past, mm(a, b.t()) * scale, -math.inf), 1)
        size = torch.where(past, mm(a.abs(), b.abs().t()) * scale, 0.0).amax(1, keepdim=True)
        E = (d + 16) * U * (size + 16) + (L + 16) * U
        out = mm(w, c)
        t_out = ((H + 2 * E + (L + 8) * U) * mm(w, c.abs()) + L * S * c.abs().amax() + H * out.abs() + S)
        p, p_size = mm(g, c.t()), mm(g.abs(), c.abs().t())
        delta = (g * out).sum(1, keepdim=True)
        t_delta = (g.abs() * t_out).sum(1, keepdim=True) + (d + 8) * U * (g * out).abs().sum(1, keepdim=True)
        few = w * (E * p.abs() + (d + 8) * U * p_size) + (summed + 16) * U * (w * p).abs()
        t_delta[:summed] = few.sum(1, keepdim=True)[:summed]
        x = w * (p - delta)
        t_w = torch.where(past, (H + E) * w + 2.0**-39, 0.0)
        t_x = torch.where(past, w * (E * (p - delta).abs() + (d + 8) * U * p_size + t_delta) + H * x.abs() + 2.0**-40 * bound, 0.0)
        many = (L * rep + 8) * U
        dq[:, i], tq[:, i] = mm(x, b) * scale, (mm(t_x, b.abs()) + many * mm(x.abs(), b.abs())) * scale
        dk[:, i // rep] += mm(x.t(), a) * scale
        tk[:, i // rep] += (mm(t_x.t(), a.abs()) + many * mm(x.abs().t(), a.abs())) * scale
        dv[:, i // rep] += mm(w.t(), g)
        tv[:, i // rep] += mm(t_w.t(), g.abs()) + many * mm(w.t(), g.abs())
    return (dq, dk, dv), tuple(t + H * r.abs() + S for t, r in ((tq, dq), (tk, dk), (tv, dv)))


def make(r, total, n, g, d, fused, device, spread=1.0, e_spread=1.0):
    sizes = (n, g, g)
    new = lambda *shape, by=spread: torch.from_numpy((r.standard_normal(shape) * by).astype(np.float16)).to(device)
    if fused:
        q, k, v = new(total, sum(sizes), d).split(sizes, dim=1)
    else:
        q, k, v = (new(total, s, d) for s in sizes)
    return q, k, v, new(total, n, d, by=e_spread)


def starts_of(lengths, device, first=0):
    return torch.tensor([first] + [first + int(x) for x in np.cumsum(lengths)], dtype=torch.int64, device=device)


def grads(K, q, k, v, e, starts, scale=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = K.flash_attention_packed(*leaves, starts, scale=scale)
    return (out, *torch.autograd.grad(out, leaves, e))


def check(K, q, k, v, e, lengths, scale=None, first=0):
    starts = starts_of(lengths, q.device, first)
    out, *got = grads(K, q, k, v, e, starts, scale)
    assert torch.equal(out[first:first + sum(lengths)],
                       K.flash_attention_packed(q, k, v, starts, scale=scale)[first:first + sum(lengths)])
    for x, like in zip(got, (q, k, v)):
        assert x.shape == like.shape and x.dtype == torch.float16 and x.is_contiguous()
    bound = largest_norm(e) * largest_norm(v)
    at = first
    for L in lengths:
        rows = slice(at, at + L)
        at += L
        if L:
            w, tol = want(q[rows], k[rows], v[rows], e[rows], q.shape[2] ** -0.5 if scale is None else scale, bound)
            for name, x, y, t in zip("qkv", got, w, tol):
                off = (x[rows].double() - y).abs()
                assert torch.all(off <= t), (name, L, float((off / t).max()))
    for x in got:
        assert not x[:first].any() and not x[at:].any()
    return got


LENGTHS = [[1], [2], [31], [32, 33], [63, 64, 65], [127, 1, 128, 129], [0, 5, 0, 0, 257, 1, 0], [191, 320, 640, 7],
           [1] * 40, [1000, 1, 383]]


@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads", [(12, 12), (8, 2), (25, 25)])
@pytest.mark.parametrize("fused", [True, False])
def test_lengths(K, gpu_device, d, heads, fused):
    r = np.random.default_rng(d)
    for lengths in LENGTHS:
        if heads[0] == 25 and sum(lengths) > 400:
            continue
        check(K, *make(r, sum(lengths), *heads, d, fused, gpu_device), lengths)


@pytest.mark.parametrize("d", [16, 64, 128, 256])
@pytest.mark.parametrize("heads", [(1, 1), (7, 7), (9, 9), (32, 8), (6, 1), (36, 9), (64, 16)])
def test_heads(K, gpu_device, d, heads):
    r = np.random.default_rng(heads[0])
    lengths = [150, 64, 3, 97]
    check(K, *make(r, sum(lengths), *heads, d, True, gpu_device), lengths)


@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
def test_many_blocks(K, gpu_device, d):
    """Few sequences and blocks, whose heaviest come first, and many."""
    r = np.random.default_rng(19)
    for heads, lengths in (((20, 20), [65, 1000, 129, 0, 640, 1300]), ((48, 12), r.integers(0, 30, 300).tolist()),
                           ((64, 8), [1] * 200 + [100, 200])):
        check(K, *make(r, sum(lengths), *heads, d, True, gpu_device), lengths)


@pytest.mark.parametrize("d", [16, 64, 256])
@pytest.mark.parametrize("first,behind", [(0, 9), (5, 0), (70, 130)])
def test_rows_of_no_sequence(K, gpu_device, d, first, behind):
    r = np.random.default_rng(2)
    lengths = [40, 0, 100]
    q, k, v, e = make(r, first + sum(lengths) + behind, 4, 2, d, False, gpu_device)
    for t in (q, k, v, e):
        t[:first] = math.nan
        t[first + sum(lengths):] = math.inf
    got = check(K, q, k, v, e, lengths, first=first)
    assert all(torch.isfinite(x).all() for x in got)


@pytest.mark.parametrize("d,scale", [(64, 1.0), (64, 3.0), (128, 1e-3), (32, 40.0), (16, 1e-6)])
def test_scales(K, gpu_device, d, scale):
    r = np.random.default_rng(3)
    lengths = [130, 77]
    check(K, *make(r, sum(lengths), 4, 4, d, True, gpu_device), lengths, scale=scale)


@pytest.mark.parametrize("d", [16, 64, 128, 256])
@pytest.mark.parametrize("spread", [1e-6, 1e-3, 1.0, 1e3])
def test_sizes_of_the_output_gradient(K, gpu_device, d, spread):
    """Far below and above one, as a loss without and with a scale leaves it."""
    r = np.random.default_rng(4)
    lengths = [200, 33]
    check(K, *make(r, sum(lengths), 4, 2, d, True, gpu_device, e_spread=spread), lengths)


@pytest.mark.parametrize("d", [64, 128])
def test_rows_of_different_sizes(K, gpu_device, d):
    """Texts that count a millionth of others, some for nothing."""
    r = np.random.default_rng(5)
    lengths = [100, 150, 60]
    q, k, v, e = make(r, sum(lengths), 4, 4, d, True, gpu_device)
    e *= torch.tensor([1e-3, 1000.0, 0.0], device=gpu_device).repeat_interleave(torch.tensor(lengths, device=gpu_device))[
        :, None, None].half()
    check(K, q, k, v, e, lengths)


@pytest.mark.parametrize("d", [16, 64, 256])
def test_scores_of_thousands(K, gpu_device, d):
    """Rows whose logarithm fp32 rounds by more than fp16's step are done with the statistic itself: the softmax has one
    key of weight 1, and the gradients of q and k vanish."""
    r = np.random.default_rng(6)
    L = 70
    q, k, v, e = make(r, L, 2, 2, d, False, gpu_device)
    scale = 1e6
    out, dq, dk, dv = grads(K, q, k, v, e, starts_of([L], gpu_device), scale)
    for h in range(2):
        s = torch.mm(q[:, h].double(), k[:, h].double().t().contiguous())
        s = torch.where(torch.ones_like(s).tril_() > 0, s, -math.inf)
        top2 = s.topk(2, 1)
        # fp32 sums tell them apart by far, so weights of other keys are 0
        clear = (top2.values[:, 0] - top2.values[:, 1]) * scale > 200 + 2 * (d + 16) * U * scale * d * 16
        assert clear.sum() > L - 8
        for i in torch.nonzero(clear)[:, 0].tolist():
            best = int(top2.indices[i, 0])
            # the output's weight is rounded to fp16, its denominator is not
            assert torch.all((out[i, h] - v[best, h]).double().abs() <= 2 * H * v[best, h].double().abs() + S)
        if bool(clear.all()):
            ref = torch.zeros(L, d, dtype=torch.float64, device=gpu_device).index_add_(0, top2.indices[:, 0], e[:, h].double())
            assert torch.all((dv[:, h].double() - ref).abs() <= (H + L * U) * ref.abs() + S + 1e-5)
    assert torch.isfinite(dq).all() and torch.isfinite(dk).all() and torch.isfinite(dv).all()


def sparse_want(q, k, v, e, scale):
    """Row by row, so that a hidden row takes no part whatever it holds; [L, d] in 64 bits on the CPU."""
    L = q.shape[0]
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i in range(L):
        kk, vv = k[:i + 1], v[:i + 1]
        w = torch.softmax(kk @ q[i] * scale, 0)
        p = vv @ e[i]
        x = w * (p - (w * p).sum()) * scale
        dq[i] = x @ kk
        dk[:i + 1] += x[:, None] * q[i]
        dv[:i + 1] += w[:, None] * e[i]
    return dq, dk, dv


@pytest.mark.parametrize("d", [16, 64, 128, 256])
@pytest.mark.parametrize("which", [0, 1, 2, 3])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_what_hidden_rows_hold(K, gpu_device, d, which, value):
    """A NaN or an infinity in one row spoils the gradients that the formula says, and no others."""
    r = np.random.default_rng(7)
    lengths = [90, 40]
    bad = 37
    t = list(make(r, sum(lengths), 2, 1, d, False, gpu_device))
    t[which][bad, -1, 3] = value
    out, *got = grads(K, *t, starts_of(lengths, gpu_device))
    q, k, v, e = (x.double().cpu() for x in t)
    clean = list(make(np.random.default_rng(7), sum(lengths), 2, 1, d, False, gpu_device))
    bound = largest_norm(clean[3]) * largest_norm(clean[2])
    for rows in (slice(0, 90), slice(90, 130)):
        ref = [torch.zeros(rows.stop - rows.start, n, d, dtype=torch.float64) for n in (2, 1, 1)]
        for h in range(2):
            for x, y in zip(ref, sparse_want(q[rows, h], k[rows, 0], v[rows, 0], e[rows, h], d**-0.5)):
                x[:, h if x.shape[1] == 2 else 0] += y
        _, tol = want(*(x[rows] for x in clean), d**-0.5, bound)
        for x, y, limit in zip(got, ref, tol):
            x, fine = x[rows].double().cpu(), torch.isfinite(y)
            assert torch.equal(torch.isfinite(x), fine)
            # without the spoilt row the sums have fewer terms: the clean ones' tolerance twice, and its own row's part
            assert torch.all((x - y).abs()[fine] <= 2 * limit.cpu()[fine] + H * y.abs()[fine])


def test_large_gradients_are_finite(K, gpu_device):
    """u would pass fp16's range, the gradients do not."""
    r = np.random.default_rng(8)
    q, k, v, e = make(r, 100, 2, 2, 64, False, gpu_device)
    q, k, v, e = q * 1e-3, k * 1e-3, v * 300, e * 30
    check(K, q, k, v, e, [100])


@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
def test_first_rows(K, gpu_device, d):
    """A query with one key has weight 1 whatever its score is: its gradient is 0, and so is what it adds to the key's."""
    r = np.random.default_rng(15)
    lengths = [1] * 70
    q, k, v, e = make(r, 70, 4, 2, d, True, gpu_device)
    _, dq, dk, dv = grads(K, q, k, v, e, starts_of(lengths, gpu_device))
    assert not dq.any() and not dk.any()
    assert torch.equal(dv, (e[:, 0::2].float() + e[:, 1::2].float()).half())
    _, dq, dk, dv = grads(K, q, k, v, e, starts_of([30, 40], gpu_device))
    assert not dq[0].any() and not dq[30].any() and dq[1:30].any() and dq[31:].any()


def test_same_bits(K, gpu_device):
    r = np.random.default_rng(9)
    lengths = [300, 1, 513]
    q, k, v, e = make(r, sum(lengths), 8, 2, 64, True, gpu_device)
    starts = starts_of(lengths, gpu_device)
    first = grads(K, q, k, v, e, starts)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, grads(K, q, k, v, e, starts)))


def test_some_of_the_gradients(K, gpu_device):
    r = np.random.default_rng(10)
    q, k, v, e = make(r, 80, 4, 2, 64, True, gpu_device)
    starts = starts_of([50, 30], gpu_device)
    _, *every = grads(K, q, k, v, e, starts)
    for need in ((True, False, False), (False, True, False), (False, False, True), (True, False, True)):
        leaves = [t.detach().requires_grad_(n) for t, n in zip((q, k, v), need)]
        out = K.flash_attention_packed(*leaves, starts)
        got = torch.autograd.grad(out, [t for t in leaves if t.requires_grad], e)
        assert all(torch.equal(a, b) for a, b in zip(got, [g for g, n in zip(every, need) if n]))
    with torch.no_grad():
        assert not K.flash_attention_packed(*[t.detach().requires_grad_() for t in (q, k, v)], starts).requires_grad
    buf = torch.empty_like(out)
    assert not K.flash_attention_packed(*[t.detach().requires_grad_() for t in (q, k, v)], starts, out=buf).requires_grad


def test_forms_of_the_output_gradient(K, gpu_device):
    """One number for all of it, as a sum hands it on, columns of something wider, an odd address."""
    r = np.random.default_rng(11)
    q, k, v, e = make(r, 80, 4, 2, 64, True, gpu_device)
    starts = starts_of([50, 30], gpu_device)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    one = torch.autograd.grad(K.flash_attention_packed(*leaves, starts).float().sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(one, grads(K, q, k, v, torch.ones_like(e), starts)[1:]))
    wide = torch.zeros(80, 7, 72, dtype=torch.float16, device=gpu_device)
    wide[:, 1:5, 4:68] = e
    odd = torch.zeros(e.numel() + 1, dtype=torch.float16, device=gpu_device)[1:].view(e.shape)
    odd.copy_(e)
    every = grads(K, q, k, v, e, starts)
    for x in (wide[:, 1:5, 4:68], odd):
        assert all(torch.equal(a, b) for a, b in zip(every, grads(K, q, k, v, x, starts)))


def test_through_a_product(K, gpu_device):
    """q, k and v as the columns of a leaf: its gradient has all three."""
    r = np.random.default_rng(12)
    y = torch.from_numpy(r.standard_normal((90, 8, 64)).astype(np.float16)).to(gpu_device).requires_grad_()
    e = torch.from_numpy(r.standard_normal((90, 4, 64)).astype(np.float16)).to(gpu_device)
    starts = starts_of([60, 30], gpu_device)
    K.flash_attention_packed(*y.split((4, 2, 2), dim=1), starts).backward(e)
    parts = grads(K, *y.detach().split((4, 2, 2), dim=1), e, starts)[1:]
    assert torch.equal(y.grad, torch.cat(parts, dim=1))


def test_derivatives_that_there_are_not(K, gpu_device):
    q = torch.randn(8, 2, 64, device=gpu_device).half().requires_grad_()
    starts = starts_of([8], gpu_device)
    out = K.flash_attention_packed(q, q, q, starts)
    with pytest.raises(RuntimeError, match="first derivative"):
        torch.autograd.grad(out.float().sum(), q, create_graph=True)


def test_nothing(K, gpu_device):
    q = torch.zeros(0, 2, 64, dtype=torch.float16, device=gpu_device).requires_grad_()
    out = K.flash_attention_packed(q, q, q, torch.tensor([0, 0], device=gpu_device))
    out.sum().backward()
    assert q.grad.shape == q.shape
    q = torch.full((4, 2, 64), math.nan, dtype=torch.float16, device=gpu_device).requires_grad_()
    out = K.flash_attention_packed(q, q, q, torch.tensor([2, 2], device=gpu_device))
    out.backward(torch.full_like(out, math.nan))
    assert not q.grad.any()


def test_other_stream(K, gpu_device):
    r = np.random.default_rng(13)
    q, k, v, e = make(r, 300, 4, 4, 64, True, gpu_device)
    starts = starts_of([300], gpu_device)
    every = grads(K, q, k, v, e, starts)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = grads(K, q, k, v, e, starts)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(every, got))


def test_captured_step(K, gpu_device):
    """Captured once, replayed for other values and other lengths, eager work between the replays."""
    r = np.random.default_rng(14)
    lengths = ([200, 56], [1, 255], [100, 156])
    q, k, v, e = make(r, 256, 4, 2, 64, False, gpu_device)
    starts = starts_of(lengths[0], gpu_device)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]

    def step():
        out = K.flash_attention_packed(*leaves, starts)
        return (out, *torch.autograd.grad(out, leaves, e))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n, some in enumerate(lengths):
        new = make(np.random.default_rng(20 + n), 256, 4, 2, 64, False, gpu_device)
        with torch.no_grad():
            for t, x in zip((*leaves, e), new):
                t.copy_(x)
        starts.copy_(starts_of(some, gpu_device))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, grads(K, *new, starts_of(some, gpu_device))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads", [(4, 4), (8, 1)])
def test_some_of_the_gradients_of_every_size(K, gpu_device, d, heads):
    """Each walk in a launch of its own, and the heads over a key head divided or not."""
    r = np.random.default_rng(16)
    lengths = [150, 1, 70]
    q, k, v, e = make(r, 221, *heads, d, True, gpu_device)
    starts = starts_of(lengths, gpu_device)
    _, *every = grads(K, q, k, v, e, starts)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        leaves = [t.detach().requires_grad_(n) for t, n in zip((q, k, v), need)]
        got = torch.autograd.grad(K.flash_attention_packed(*leaves, starts), [t for t in leaves if t.requires_grad], e)
        assert all(torch.equal(a, b) for a, b in zip(got, [g for g, n in zip(every, need) if n]))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("far_heads", [False, True])
def test_offsets_beyond_32_bits(K, gpu_device, d, far_heads):
    """Rows, or heads, so far apart that their offsets pass 2^32 bytes: the gradients of dense copies."""
    r = np.random.default_rng(17)
    dense = make(r, 140, 4, 2, d, False, gpu_device)
    starts = starts_of([5, 135], gpu_device)
    far = []
    if far_heads:
        wide = torch.empty(4, 1 << 30, dtype=torch.float16, device=gpu_device)
        for n, t in enumerate(dense[:3]):
            far.append(wide[:t.shape[1], n << 20:(n << 20) + 140 * d].view(t.shape[1], 140, d).transpose(0, 1))
    else:
        wide = torch.empty(140, 1 << 24, dtype=torch.float16, device=gpu_device)
        for n, t in enumerate(dense[:3]):
            at = (1 << 24) - (n + 1) * 1024
            far.append(wide[:, at:at + t.shape[1] * d].view(140, t.shape[1], d))
    for x, t in zip(far, dense):
        x.copy_(t)
    assert all(torch.equal(a, b) for a, b in zip(grads(K, *far, dense[3], starts), grads(K, *dense, starts)))


def test_two_streams_at_once(K, gpu_device):
    r = np.random.default_rng(18)
    lengths = [700, 300]
    inputs = [make(r, 1000, 8, 2, 128, True, gpu_device) for _ in range(2)]
    starts = starts_of(lengths, gpu_device)
    alone = [grads(K, *t, starts) for t in inputs]
    sides = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for n, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[n].append(grads(K, *inputs[n], starts))
    torch.cuda.synchronize()
    for n in range(2):
        for one in got[n]:
            assert all(torch.equal(a, b) for a, b in zip(one, alone[n]))


def test_two_graphs_with_one_pool(K, gpu_device):
    """Replayed by turns: each result stands until its own graph, or one that shares its memory, runs again."""
    r = np.random.default_rng(20)
    inputs = [make(r, 200, 4, 1, 64, False, gpu_device) for _ in range(2)]
    starts = [starts_of(x, gpu_device) for x in ([120, 80], [3, 197])]
    leaves = [[t.detach().requires_grad_() for t in x[:3]] for x in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads(K, *inputs[0], starts[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, got = [], []
    for n in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            out = K.flash_attention_packed(*leaves[n], starts[n])
            got.append((out, *torch.autograd.grad(out, leaves[n], inputs[n][3])))
        graphs.append(graph)
    for turn in range(3):
        for n in range(2):
            with torch.no_grad():
                inputs[n][3].mul_(-1)
            graphs[n].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got[n], grads(K, *inputs[n], starts[n])))


def test_what_is_changed_behind_the_forward_pass(K, gpu_device):
    """torch's versions: what the gradients need may not be written in between."""
    r = np.random.default_rng(21)
    for which in range(3):
        q, k, v, e = make(r, 30, 2, 2, 64, False, gpu_device)
        starts = starts_of([30], gpu_device)
        q.requires_grad_()
        out = K.flash_attention_packed(q, k, v, starts)
        with torch.no_grad():
            (k, v, starts)[which].add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward(e)


@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads", [(12, 12), (8, 2), (7, 1)])
def test_deltas_of_the_first_queries(K, gpu_device, d, heads):
    """Of the first 16 queries what the output is rounded by plays no part."""
    r = np.random.default_rng(23)
    lengths = [16, 2, 3, 0, 9, 15, 1, 12, 5, 16]
    q, k, v, e = make(r, sum(lengths) + 3, *heads, d, True, gpu_device)
    starts = starts_of(lengths, gpu_device, 2)
    _, *got = grads(K, q, k, v, e, starts)
    bound, at = largest_norm(e) * largest_norm(v), 2
    for L in lengths:
        rows = slice(at, at + L)
        at += L
        if L:
            w, tol = want(q[rows], k[rows], v[rows], e[rows], d**-0.5, bound, summed=16)
            for name, x, y, t in zip("qkv", got, w, tol):
                off = (x[rows].double() - y).abs()
                assert torch.all(off <= t), (name, L, float((off / t).max()))


def test_first_queries_of_many_sequences(K, gpu_device):
    """More sequences and heads than wavefronts of the launch for the first queries."""
    r = np.random.default_rng(24)
    n, L = 10000, 3
    q, k, v, e = make(r, n * L, 32, 4, 16, False, gpu_device)
    _, *got = grads(K, q, k, v, e, starts_of([L] * n, gpu_device))
    some = [0, 1, 8191, 8192, 9999]
    for s in some:
        rows = slice(s * L, s * L + L)
        w, tol = want(q[rows], k[rows], v[rows], e[rows], 0.25, largest_norm(e) * largest_norm(v), summed=16)
        for x, y, t in zip(got, w, tol):
            assert torch.all((x[rows].double() - y).abs() <= t)
