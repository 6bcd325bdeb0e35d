"""token_log_probs and distillation_loss on the GPU against their formulas in 64 bits.

Tolerances, from the arithmetic (u = 2^-24, half a step of fp32):
  * a term exp((x - m) / tau) is off by 4 u + 3 u |x - m| / tau relative: the scaled difference is rounded three
    times, the hardware's exponential is within a step.  Terms far below the maximum are off by more and weigh less: t exp(-t)
    is at most 0.37, so in a sum they count for 2 u at most;
  * a sum of V terms by at least 256 threads is off by at most ceil(V / 256) + 16 additions, u each, relative (all
    terms have one sign): SUM(V) = u (8 + ceil(V / 256) + 16);
  * a log probability is a scaled difference, off by 3 u relative, less a logarithm, off by SUM(V) and 4 u relative;
  * an entropy is the sum of two numbers of one sign, each a quotient or logarithm of such sums whose terms e t are
    off by the 4 u + 3 u t of e: 64 u + 2 SUM(V) relative, which covers t up to 19 for every term and, weighed,
    all above;
  * a gradient's parts are products of such numbers: 100 u + 2 SUM(V) of each part's size, added without
    cancelling, and half a step of the storage type for the result (of subnormal numbers: half the smallest)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
DTYPES = [torch.float16, torch.float32]


@pytest.fixture(scope="module")
def K(gpu_device):
    from gpt_triton_amd import kernels

    return kernels


def sum_error(V):
    return U * (8 + -(-V // 256) + 16)


def storage(d, dtype):
    return np.abs(d) * torch.finfo(dtype).eps / 2 + (2.0**-25 if dtype == torch.float16 else 2.0**-149)


def on_gpu(x, dtype, device, offset=0, pitch=None):
    """x [rows, V] as a view of rows at `pitch`, `offset` elements into the allocation; NaN around them."""
    rows, V = x.shape
    pitch = pitch or V
    buf = torch.full((offset + rows * pitch + 16,), math.nan, dtype=dtype, device=device)
    view = buf.as_strided((rows, V), (pitch, 1), offset)
    view.copy_(torch.from_numpy(np.ascontiguousarray(x)).to(dtype))
    return view


def crowd(r, rows, V, spread=2.5):
    x = r.standard_normal((rows, V)) * spread
    at = r.integers(0, V, size=(rows, min(V, 4)))
    np.put_along_axis(x, at, r.uniform(0, 15, at.shape), 1)
    return x


def log_softmax(x, tau):
    z = x.astype(np.float64) / tau
    m = z.max(1, keepdims=True)
    m = np.where(np.isfinite(m), m, 0.0)
    with np.errstate(divide="ignore", invalid="ignore"):
        return z - m - np.log(np.exp(z - m).sum(1, keepdims=True))


def want_scores(x, tokens, tau):
    z = log_softmax(x, tau)
    p = np.exp(z)
    lp = np.where((tokens >= 0) & (tokens < x.shape[1]),
                  np.take_along_axis(z, np.clip(tokens, 0, x.shape[1] - 1)[:, None], 1)[:, 0], 0.0)
    with np.errstate(invalid="ignore"):
        return z, p, lp, -np.where(p == 0, 0.0, p * z).sum(1)


def top_ids(x, k):
    """The k largest of each row, equal ones by index."""
    return np.argsort(-x, axis=1, kind="stable")[:, :k]


def host(t):
    return t.detach().cpu().numpy()


def check_scores(K, view, tokens, top, tau=1.0):
    x = host(view).astype(np.float64)
    V = x.shape[1]
    z, p, lp, ent = want_scores(x, tokens, tau)
    r = K.token_log_probs(view, torch.from_numpy(tokens).to(view.device), top=top, temperature=tau)
    d = np.abs(np.take_along_axis(x, np.clip(tokens, 0, V - 1)[:, None], 1)[:, 0] - x.max(1)) / tau
    tol = U * 3 * d + sum_error(V) + 4 * U * np.abs(lp)
    # the likeliest token's is a logarithm near 1, and keeps its relative exactness
    tol = np.where(d == 0, (sum_error(V) + 8 * U) * np.abs(lp) + 2.0**-149, tol)
    assert np.all(np.abs(host(r.log_probs) - lp) <= tol), np.max(np.abs(host(r.log_probs) - lp) / tol)
    tol = (64 * U + 2 * sum_error(V)) * ent + 1e-37
    assert np.all(np.abs(host(r.entropy) - ent) <= tol), np.max(np.abs(host(r.entropy) - ent) / tol)
    if top == 0:
        assert r.top_tokens is None and r.top_log_probs is None
        return
    ids = top_ids(x, top)
    assert np.array_equal(host(r.top_tokens), ids)
    want = np.take_along_axis(z, ids, 1)
    # lowest less highest, -6.8e38, is no fp32 number (the largest is 3.4e38): it rounds to -infinity
    want = np.where(want < -float(np.finfo(np.float32).max), -math.inf, want)
    got = host(r.top_log_probs)
    same = np.isneginf(want) & np.isneginf(got)
    d = (x.max(1)[:, None] - np.take_along_axis(x, ids, 1)) / tau
    with np.errstate(invalid="ignore"):
        err = np.where(same, 0.0, np.abs(got - want))
        assert np.all(err <= np.where(same, 0.0, U * 3 * d + sum_error(V) + 4 * U * np.abs(want)))


SIZES = [1, 2, 7, 8, 9, 63, 300, 2047, 2049, 4097, 8193, 20000, 32000, 50257, 50304, 65024, 81921, 131072, 163841, 200003]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", SIZES)
def test_scores(K, gpu_device, dtype, V):
    r = np.random.default_rng(V)
    for rows, offset, pitch, tau in ((3, 0, None, 1.0), (2, 1, V + 3, 0.7), (1, 5, None, 2.0)):
        view = on_gpu(crowd(r, rows, V), dtype, gpu_device, offset, pitch)
        tokens = r.integers(0, V, size=rows)
        tokens[0] = host(view)[0].argmax()
        for top in {0, 1, min(V, 5), min(V, 16), min(V, 17), min(V, 128)}:
            check_scores(K, view, tokens, top, tau)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [257, 1477])
def test_many_rows(K, gpu_device, dtype, rows):
    r = np.random.default_rng(rows)
    view = on_gpu(crowd(r, rows, 1537), dtype, gpu_device, 0, 1600)
    check_scores(K, view, r.integers(0, 1537, size=rows), 20)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [300, 5000, 50257, 200003])
@pytest.mark.parametrize("top", [1, 7, 16, 40, 128])
def test_equal_logits_come_in_order(K, gpu_device, dtype, V, top):
    r = np.random.default_rng(top)
    few = r.integers(0, 3, size=(1, V)).astype(np.float64)
    owners = np.where((np.arange(V) // 8) % 256 < 6, 5.0 + r.random(V), r.random(V))[None]  # the largest with few threads
    steps = np.floor(r.standard_normal((1, V)) * 8) / 8
    signs = np.where(r.random((1, V)) < 0.5, 0.0, -0.0)
    for x in (np.zeros((1, V)), few, owners, steps, signs, np.arange(V)[None] % 7.0, -np.arange(V)[None] / 64.0):
        check_scores(K, on_gpu(x, dtype, gpu_device, 3), np.array([V // 2]), top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [9, 300, 50257, 200003])
def test_masked_logits(K, gpu_device, dtype, V):
    """Tokens that cannot occur, as -infinity and as the type's lowest value."""
    r = np.random.default_rng(V)
    for hidden in (-math.inf, float(torch.finfo(dtype).min)):
        for kept in (1, 3, V // 2):
            x = crowd(r, 1, V)
            keep = r.permutation(V)[:kept]
            y = np.full_like(x, hidden)
            y[0, keep] = x[0, keep]
            check_scores(K, on_gpu(y, dtype, gpu_device, 1), keep[:1], min(V, 5))
    # all of them the lowest value: an even distribution
    check_scores(K, on_gpu(np.full((2, V), float(torch.finfo(dtype).min)), dtype, gpu_device), np.array([0, V - 1]), 2)
    # the widest range that the type has: differences beyond it
    x = np.full((1, V), float(torch.finfo(dtype).min))
    x[0, V // 3] = float(torch.finfo(dtype).max)
    check_scores(K, on_gpu(x, dtype, gpu_device), np.array([V // 3]), 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [5, 300, 50257, 200003])
def test_rows_without_any_probability(K, gpu_device, dtype, V):
    x = torch.full((2, V), -math.inf, dtype=dtype, device=gpu_device)
    x[1] = 0.0
    t = torch.tensor([V - 1, V - 1], device=gpu_device)
    r = K.token_log_probs(x, t, top=3)
    assert host(r.log_probs)[0] == -math.inf and host(r.entropy)[0] == 0.0
    assert host(r.top_tokens).tolist() == [[0, 1, 2]] * 2
    assert np.all(np.isneginf(host(r.top_log_probs)[0])) and np.all(np.isfinite(host(r.top_log_probs)[1]))
    x.requires_grad_()
    r = K.token_log_probs(x, t, top=3)
    grad, = torch.autograd.grad((r.log_probs.sum() + r.entropy.sum() + r.top_log_probs[1].sum(),), x)
    assert torch.all(grad[0] == 0) and torch.all(torch.isfinite(grad[1]))
    loss, grad = K.distillation_loss_and_grad(x, t[:, None], torch.zeros(2, 1, device=gpu_device))
    assert host(loss)[0] == math.inf and np.isfinite(host(loss)[1]) and torch.all(grad[0] == 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [300, 50257, 200003])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_numbers_that_are_none(K, gpu_device, dtype, V, bad):
    """A NaN or an infinity spoils its row and no other, and the top tokens stay tokens."""
    r = np.random.default_rng(5)
    x = crowd(r, 3, V)
    x[1, [0, V // 2, V - 1]] = bad
    view = on_gpu(x, dtype, gpu_device)
    tokens = torch.tensor([1, 1, 1], device=gpu_device)
    s = K.token_log_probs(view, tokens, top=128)
    for out in (s.log_probs, s.entropy, s.top_log_probs.sum(1)):
        assert np.array_equal(np.isnan(host(out)), [False, True, False])
    ids = host(s.top_tokens)
    clean = host(view).astype(np.float64)
    clean[np.isnan(clean)] = -math.inf
    assert np.array_equal(ids, top_ids(clean, 128))
    loss, grad = K.distillation_loss_and_grad(view, s.top_tokens, torch.zeros(3, 128, device=gpu_device))
    assert np.array_equal(np.isnan(host(loss)), [False, True, False])
    assert torch.all(torch.isfinite(grad[0::2])) and torch.any(torch.isnan(grad[1]))
    # as padding they do nothing
    weights = torch.tensor([1.0, 0.0, 1.0], device=gpu_device)
    loss, grad = K.distillation_loss_and_grad(view, s.top_tokens, torch.zeros(3, 128, device=gpu_device), 1.0, weights)
    assert np.all(np.isfinite(host(loss))) and torch.all(grad[1] == 0) and torch.all(torch.isfinite(grad))
    view.requires_grad_()
    lp = K.token_log_probs(view, torch.tensor([1, -100, 1], device=gpu_device)).log_probs
    grad, = torch.autograd.grad(lp.sum(), view)
    assert np.all(np.isfinite(host(lp))) and torch.all(torch.isfinite(grad[0::2]))


def test_tokens_outside_the_vocabulary(K, gpu_device):
    x = on_gpu(crowd(np.random.default_rng(1), 5, 777), torch.float16, gpu_device)
    x.requires_grad_()
    t = torch.tensor([-100, -1, 777, 2**40, 5], device=gpu_device)
    lp = K.token_log_probs(x, t).log_probs
    assert torch.all(lp[:4] == 0) and lp[4] < 0
    grad, = torch.autograd.grad(lp.sum(), x)
    assert torch.all(grad[:4] == 0) and torch.any(grad[4] != 0)


def want_score_gradient(x, tokens, tau, g, h, ids, u):
    """(gradient, sizes of its parts added up)."""
    z, p, _, ent = want_scores(x, tokens, tau)
    one = np.zeros_like(p)
    size = np.zeros_like(p)
    inside = (tokens >= 0) & (tokens < x.shape[1])
    g = np.where(inside, g, 0.0)
    rows = np.arange(len(p))
    np.add.at(one, (rows[inside], tokens[inside]), g[inside])
    np.add.at(size, (rows[inside], tokens[inside]), np.abs(g[inside]))
    for i in range(ids.shape[1]):
        np.add.at(one, (rows, ids[:, i]), u[:, i])
        np.add.at(size, (rows, ids[:, i]), np.abs(u[:, i]))
    zz = np.where(p == 0, 0.0, z)
    total = (g + u.sum(1))[:, None]
    d = one - p * (total + h[:, None] * (zz + ent[:, None]))
    size = size + p * ((np.abs(g) + np.abs(u).sum(1))[:, None] + np.abs(h)[:, None] * (np.abs(zz) + ent[:, None]))
    return d / tau, size / tau


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 9, 300, 2049, 50257, 50304, 131072, 200003])
@pytest.mark.parametrize("parts", ["token", "entropy", "top", "all"])
def test_score_gradients(K, gpu_device, dtype, V, parts):
    r = np.random.default_rng(V)
    for rows, offset, pitch, tau in ((4, 0, None, 1.0), (2, 1, V + 7, 0.7)):
        x = crowd(r, rows, V)
        if V > 300:
            x[:, r.permutation(V)[:V // 5]] = -math.inf
        view = on_gpu(x, dtype, gpu_device, offset, pitch).requires_grad_()
        x = host(view).astype(np.float64)
        top = min(V, 20)
        tokens = top_ids(x, 1)[:, 0]  # the token is one of the top ones: two parts meet
        tokens[-1] = r.integers(0, V) if V <= 300 else top_ids(x, 40)[-1, -1]
        g, h, u = (r.standard_normal(s).astype(np.float32) for s in (rows, rows, (rows, top)))
        s = K.token_log_probs(view, torch.from_numpy(tokens).to(gpu_device), top=top, temperature=tau)
        outs, grads = [], []
        for name, out, w in (("token", s.log_probs, g), ("entropy", s.entropy, h), ("top", s.top_log_probs, u)):
            if parts in (name, "all"):
                outs.append(out)
                grads.append(torch.from_numpy(w).to(gpu_device))
            else:
                w[:] = 0
        got, = torch.autograd.grad(outs, view, grads)
        assert got.shape == view.shape and got.dtype == dtype
        d, size = want_score_gradient(x, tokens, tau, g.astype(np.float64), h.astype(np.float64), host(s.top_tokens),
                                      u.astype(np.float64))
        tol = (100 * U + 2 * sum_error(V)) * size + storage(d, dtype)
        err = np.abs(host(got).astype(np.float64) - d)
        assert np.all(err <= tol), np.max(err / tol)


def want_distillation(x, ids, teacher, tau, w):
    z = log_softmax(x, tau)
    p = np.exp(z)
    there = (ids >= 0) & (ids < x.shape[1])
    t = np.where(there, teacher.astype(np.float64) / tau, -math.inf)
    m = t.max(1, keepdims=True)
    e = np.exp(t - np.where(np.isfinite(m), m, 0.0))
    total = e.sum(1, keepdims=True)
    q = e / np.where(total == 0, 1.0, total)
    at = np.where(there, ids, 0)
    with np.errstate(divide="ignore", invalid="ignore"):
        terms = np.where(q == 0, 0.0, q * (np.log(q) - np.take_along_axis(z, at, 1)))
        parts = np.where(q == 0, 0.0, q * (np.abs(np.log(q)) + np.abs(np.take_along_axis(z, at, 1)) + 1))
    d = p * (total > 0)
    size = d.copy()
    for i in range(ids.shape[1]):
        rows = np.arange(len(p))
        np.add.at(d, (rows, at[:, i]), -q[:, i])
        np.add.at(size, (rows, at[:, i]), q[:, i])
    s = (w / tau)[:, None]
    return w * terms.sum(1), np.abs(w) * parts.sum(1), d * s, size * np.abs(s)


def check_distillation(K, view, ids, teacher, tau, w, what=""):
    device, dtype, V = view.device, view.dtype, view.shape[1]
    x = host(view).astype(np.float64)
    loss, size, d, d_size = want_distillation(x, ids, host(teacher), tau, w)
    ids_, w_ = torch.from_numpy(ids).to(device), torch.from_numpy(w.astype(np.float32)).to(device)
    got, grad = K.distillation_loss_and_grad(view, ids_, teacher, tau, w_)
    # K terms added, each of numbers off by a few u and a log probability
    tol = (U * (32 + ids.shape[1]) + sum_error(V)) * size + 1e-37
    assert np.all(np.abs(host(got) - loss) <= tol), (what, np.max(np.abs(host(got) - loss) / tol))
    tol = ((100 + ids.shape[1]) * U + 2 * sum_error(V)) * d_size + storage(d, dtype)
    err = np.abs(host(grad).astype(np.float64) - d)
    assert grad.shape == view.shape and np.all(err <= tol), (what, np.max(err / tol))
    # the losses alone, and torch's graph behind them, are the same numbers
    leaf = view.detach().requires_grad_()
    alone = K.distillation_loss(leaf, ids_, teacher, tau, w_)
    assert torch.equal(alone.detach(), got)
    back, = torch.autograd.grad(alone.sum(), leaf)
    assert torch.equal(back, grad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 9, 300, 2049, 50257, 50304, 131072, 200003])
def test_distillation(K, gpu_device, dtype, V):
    r = np.random.default_rng(V)
    for k, tau, offset, pitch, half in ((1, 1.0, 0, None, False), (20, 2.0, 1, V + 3, True), (64, 1.0, 0, -(-V // 64) * 64, False),
                                        (65, 0.7, 2, V + 5, True), (128, 1.0, 0, None, False)):
        view = on_gpu(crowd(r, 3, V), dtype, gpu_device, offset, pitch)
        ids = r.integers(0, V, size=(3, k))  # the same token twice too
        teacher = torch.from_numpy(r.standard_normal((3, k)) * 3).to(gpu_device, torch.float16 if half else torch.float32)
        check_distillation(K, view, ids, teacher, tau, r.uniform(0.5, 2, 3), (k, tau, offset))


def test_distillation_entries_that_count_for_nothing(K, gpu_device):
    r = np.random.default_rng(3)
    V, k = 5000, 24
    for dtype in DTYPES:
        view = on_gpu(crowd(r, 4, V), dtype, gpu_device)
        ids = r.integers(0, V, size=(4, k))
        ids[0, :5], ids[1, 3], ids[1, 4], ids[2, :] = ids[0, 0], -1, V, -100
        teacher = torch.from_numpy(r.standard_normal((4, k))).float().to(gpu_device)
        teacher[0, 7:9] = -math.inf
        teacher[3] = -math.inf
        ids[1, 5] = 2**40
        teacher[1, 3:6] = math.nan  # of no entry
        check_distillation(K, view, ids, teacher, 1.0, np.array([1.0, 1.0, 1.0, 1.0]))
        loss, grad = K.distillation_loss_and_grad(view, torch.from_numpy(ids).to(gpu_device), teacher)
        assert loss[2] == 0 and loss[3] == 0 and torch.all(grad[2:] == 0)


def test_the_least_temperature(K, gpu_device):
    """Differences of logits that are infinite when divided: all probability on the largest, and nothing that is no number.
    fp16 logits, whose exponents are off by a rounding of 60000 log2(e) / tau, have a larger least: the one probability is
    e / (e + 0) there, a quotient of two roundings, 1 / tau of it a gradient."""
    for dtype, tau in ((torch.float32, 1e-30), (torch.float16, 1e-4)):
        x = torch.zeros(2, 600, dtype=dtype, device=gpu_device)
        x[:, 7], x[:, 9] = 60000.0, -60000.0
        ids = torch.tensor([[9, 7, 11]] * 2, device=gpu_device)
        teacher = torch.tensor([[0.0, 1e30, -1e30], [-3e38, 3e38, 0.0]], device=gpu_device)
        loss, grad = K.distillation_loss_and_grad(x, ids, teacher, tau)
        assert torch.all(loss == 0) and torch.all(grad.abs() <= (0 if dtype == torch.float32 else 4 * U / tau))
        s = K.token_log_probs(x, torch.tensor([7, 7], device=gpu_device), top=1, temperature=tau)
        assert torch.all(s.log_probs == 0) and torch.all(s.entropy == 0) and torch.all(s.top_tokens == 7)
        for call in (lambda t: K.token_log_probs(x, temperature=t), lambda t: K.distillation_loss(x, ids, teacher, t)):
            with pytest.raises(ValueError):
                call(0.99 * tau)
            with pytest.raises(ValueError):
                call(1.1e30)


def test_a_teacher_that_is_the_student(K, gpu_device):
    """Scores of the whole vocabulary as the teacher: the divergence is 0 and so is the gradient, up to roundings."""
    V = 128
    x = on_gpu(crowd(np.random.default_rng(4), 6, V), torch.float32, gpu_device)
    s = K.token_log_probs(x, top=V)
    loss, grad = K.distillation_loss_and_grad(x, s.top_tokens, s.top_log_probs)
    # each of the terms q (log q - log p) is a difference of numbers up to 20 that are off by a few steps
    assert torch.all(loss.abs() <= 20 * U * 64) and torch.all(grad.abs() <= 64 * U)


def test_gradients_against_differences(K, gpu_device):
    """Central differences of the fp32 forward: step 2^-5; the third derivatives of log p, H and the loss are below 8, so the
    truncation is below 8 / 6 * 2^-10, and the forwards' roundings, 50 u, over 2^-4."""
    r = np.random.default_rng(6)
    V, step = 23, 2.0**-5
    base = np.float32(r.standard_normal(V))
    t = torch.tensor([3], device=gpu_device)
    ids = torch.from_numpy(r.integers(0, V, size=(1, 6))).to(gpu_device)
    teacher = torch.randn(1, 6, device=gpu_device)

    def values(rows):
        x = torch.from_numpy(np.float32(rows)).to(gpu_device)
        n = len(rows)
        s = K.token_log_probs(x, t.expand(n).contiguous())
        # the second of the top two as the token that it is at `base`: a step changes which one is second
        second = K.token_log_probs(x, torch.full((n,), int(top_ids(base[None], 2)[0, 1]), device=gpu_device)).log_probs
        loss = K.distillation_loss(x, ids.expand(n, -1).contiguous(), teacher.expand(n, -1).contiguous())
        return host(torch.stack((s.log_probs, s.entropy, second, loss), 1)).astype(np.float64)

    plus, minus = (values(base + sign * step * np.eye(V, dtype=np.float32)) for sign in (1, -1))
    differences = (plus - minus) / (2 * step)
    x = torch.from_numpy(base[None]).to(gpu_device).requires_grad_()
    s = K.token_log_probs(x, t, top=2)
    outs = (s.log_probs, s.entropy, s.top_log_probs[:, 1], K.distillation_loss(x, ids, teacher))
    for i, out in enumerate(outs):
        grad, = torch.autograd.grad(out.sum(), x, retain_graph=True)
        assert np.max(np.abs(host(grad)[0] - differences[:, i])) <= 8 / 6 * 2.0**-10 + 50 * U * 2**4


def test_gradients_that_come_back(K, gpu_device):
    """One number for all rows, one a row, every other one; weights of 0 whatever comes back; no second derivative."""
    r = np.random.default_rng(21)
    x = on_gpu(crowd(r, 4, 900), torch.float32, gpu_device).requires_grad_()
    ids = torch.from_numpy(r.integers(0, 900, size=(4, 6))).to(gpu_device)
    teacher = torch.from_numpy(r.standard_normal((4, 6))).float().to(gpu_device)
    w = torch.tensor([1.0, 0.0, 2.0, 0.5], device=gpu_device)
    t = ids[:, 0].contiguous()
    each = torch.tensor([3.0, math.inf, -2.0, 0.25], device=gpu_device)
    wide = torch.stack((each, each), 1)
    _, one_pass = K.distillation_loss_and_grad(x.detach(), ids, teacher, 1.0, w)
    for d in (each, wide[:, 0]):
        loss = K.distillation_loss(x, ids, teacher, 1.0, w)
        grad, = torch.autograd.grad(loss, x, d)
        assert torch.all(grad[1] == 0)
        # two products of fp32 numbers in another order: two roundings each
        want = one_pass * torch.where(w == 0, w, each)[:, None]
        assert torch.all((grad - want).abs() <= 8 * U * want.abs())
        s = K.token_log_probs(x, t)
        a, = torch.autograd.grad((s.log_probs, s.entropy), x, (d[:1].expand(4), w))
        b, = torch.autograd.grad(K.token_log_probs(x, t).log_probs, x, d[:1].expand(4).contiguous())
        c, = torch.autograd.grad(K.token_log_probs(x, t).entropy, x, w)
        assert torch.all((a - b - c).abs() <= 200 * U * (b.abs() + c.abs() + 1e-3))
    nothing = x.detach().clone()
    nothing[2] = math.nan
    nothing.requires_grad_()
    keep = torch.tensor([True, True, False, True], device=gpu_device)
    loss = torch.where(keep, K.distillation_loss(nothing, ids, teacher), 0.0)
    grad, = torch.autograd.grad(loss.sum(), nothing)
    assert torch.all(torch.isfinite(loss)) and torch.all(torch.isfinite(grad)) and torch.all(grad[2] == 0)
    loss = K.distillation_loss(x, ids, teacher)
    grad, = torch.autograd.grad(loss.sum(), x)
    assert torch.equal(grad, K.distillation_loss_and_grad(x.detach(), ids, teacher)[1])
    for out in (K.distillation_loss(x, ids, teacher), K.token_log_probs(x, t).log_probs):
        with pytest.raises(RuntimeError, match="first derivative"):
            torch.autograd.grad(out.sum(), x, create_graph=True)


def test_shapes_and_views(K, gpu_device):
    """Leading dimensions, rows of one pitch, one row many times, no rows."""
    r = np.random.default_rng(8)
    V = 700
    wide = torch.from_numpy(crowd(r, 24, 768)).half().to(gpu_device)
    flat = K.token_log_probs(wide[:, :V], torch.arange(24, device=gpu_device), top=4)
    cube = wide.view(4, 6, 768)[..., :V]
    s = K.token_log_probs(cube, torch.arange(24, device=gpu_device).view(4, 6), top=4)
    assert s.log_probs.shape == s.entropy.shape == (4, 6) and s.top_tokens.shape == (4, 6, 4)
    for a, b in zip(s, flat):
        assert torch.equal(a.flatten(), b.flatten())
    one = K.token_log_probs(wide[3, :V], torch.tensor(3, device=gpu_device), top=4)
    assert one.log_probs.shape == () and torch.equal(one.top_tokens, flat.top_tokens[3])
    assert torch.equal(one.log_probs, flat.log_probs[3])
    same = K.token_log_probs(wide[3, :V].expand(5, V), torch.arange(5, device=gpu_device))
    assert torch.all(same.entropy == flat.entropy[3])
    leaf = wide[3, :V].detach().requires_grad_()
    rows = leaf.expand(5, V)
    lp = K.token_log_probs(rows, torch.arange(5, device=gpu_device)).log_probs
    grad, = torch.autograd.grad(lp.sum(), leaf)
    assert grad.shape == (V,) and torch.all(torch.isfinite(grad))
    for empty in (wide[:0, :V], cube[:, :0]):
        s = K.token_log_probs(empty, torch.zeros(empty.shape[:-1], dtype=torch.int64, device=gpu_device), top=2)
        assert s.log_probs.shape == empty.shape[:-1] and s.top_tokens.shape == (*empty.shape[:-1], 2)
        loss, grad = K.distillation_loss_and_grad(empty, s.top_tokens, s.top_log_probs)
        assert loss.shape == empty.shape[:-1] and grad.shape == empty.shape
    column = wide[3, :V].clone().view(V, 1).t()  # a single row, whose pitch says nothing
    assert torch.equal(K.token_log_probs(column, torch.tensor([3], device=gpu_device)).log_probs[0], flat.log_probs[3])
    with pytest.raises(AssertionError):
        K.token_log_probs(wide.view(4, 6, 768)[:, :3, :V])  # rows at two pitches
    with pytest.raises(AssertionError):
        K.token_log_probs(wide.T)


def test_what_lies_between_rows_stays(K, gpu_device):
    """The gradient of the C entry writes rows and nothing between or behind them."""
    from gpt_triton_amd import _lib

    for dtype, V, pitch in ((torch.float16, 1001, 1024), (torch.float32, 50257, 50304), (torch.float16, 50257, 50259)):
        x = on_gpu(crowd(np.random.default_rng(9), 3, V), dtype, gpu_device, 0, 50304 if V > 50000 else V)
        ids = torch.zeros(3, 1, dtype=torch.int64, device=gpu_device)
        t = torch.zeros(3, 1, device=gpu_device)
        out = torch.full((3, pitch), 7.0, dtype=dtype, device=gpu_device)
        losses = torch.empty(3, device=gpu_device)
        K._call(0, "test", _lib.load().gptmi_distillation_loss, x.data_ptr(), x.stride(0), ids.data_ptr(), t.data_ptr(), 1,
                1.0, None, None, 0, losses.data_ptr(), out.data_ptr(), pitch, 3, V, K._dtype_code(x, "test"), _lib.GPTMI_F32)
        _, want = K.distillation_loss_and_grad(x, ids, t)
        assert torch.equal(out[:, :V], want) and torch.all(out[:, V:] == 7.0)


def test_rows_beyond_32_bits(K, gpu_device):
    """Rows whose elements lie past 2^31 and bytes past 2^32."""
    V, pitch = 1000, (1 << 30) + 40
    buf = torch.empty(2 * pitch + V, dtype=torch.float16, device=gpu_device)
    x = buf.as_strided((3, V), (pitch, 1))
    x.copy_(torch.from_numpy(crowd(np.random.default_rng(10), 3, V)).half())
    check_scores(K, x, np.array([1, 2, 3]), 5)
    check_distillation(K, x, np.array([[1, 2], [3, 4], [5, 6]]), torch.zeros(3, 2, device=gpu_device), 1.0, np.ones(3))


@pytest.mark.parametrize("dtype,rows", [(torch.float16, 2900), (torch.float32, 1450)])
def test_large_gradients(K, gpu_device, dtype, rows):
    """Gradients that go past the caches, from the last row on: the bits of the same rows by themselves."""
    V = 50257
    x = torch.randn(rows, 50304, device=gpu_device).mul_(2).to(dtype)[:, :V]
    ids = torch.randint(0, V, (rows, 9), device=gpu_device)
    teacher = torch.randn(rows, 9, device=gpu_device)
    w = torch.ones(rows, device=gpu_device)
    w[5] = w[-1] = 0
    d = torch.randn(rows, device=gpu_device)
    t = ids[:, 0].contiguous()

    def gradients(part):
        leaf = x[part].detach().requires_grad_()
        one, = torch.autograd.grad(K.token_log_probs(leaf, t[part]).log_probs, leaf, d[part])
        two, = torch.autograd.grad(K.distillation_loss(leaf, ids[part], teacher[part], 2.0, w[part]), leaf, d[part])
        return one, two, K.distillation_loss_and_grad(leaf, ids[part], teacher[part], 2.0, w[part])[1]

    whole = gradients(slice(0, rows))
    assert whole[0].numel() * whole[0].element_size() > 256 << 20
    for part in (slice(0, 8), slice(rows // 2, rows // 2 + 3), slice(rows - 5, rows)):
        for a, b in zip(whole, gradients(part)):
            assert torch.equal(a[part], b)
    for a in whole[1:]:
        assert torch.all(a[5] == 0) and torch.all(a[-1] == 0) and torch.all(torch.isfinite(a))


def test_millions_of_rows(K, gpu_device):
    """More workgroups than a row of the grid has: one row of logits for all of them, and rows of their own, whose chunks
    begin elsewhere: sums of another order."""
    rows, V = 2**22 + 5, 9  # four rows a workgroup
    x = torch.from_numpy(crowd(np.random.default_rng(24), 1, V)).float().to(gpu_device).expand(rows, V)
    tokens = torch.arange(rows, device=gpu_device) % V
    few = x[:V].detach().clone().requires_grad_()
    one = K.token_log_probs(few, tokens[:V])
    want, = torch.autograd.grad(one.log_probs.sum(), few, retain_graph=True)
    tol, d_tol = 2 * sum_error(V) + 40 * U, 100 * U + 2 * sum_error(V)
    s = K.token_log_probs(x, tokens)
    assert torch.all((s.log_probs - one.log_probs[tokens]).abs() <= tol)
    assert torch.all((s.entropy - one.entropy[0]).abs() <= tol + 64 * U * one.entropy[0])
    loss, grad = K.distillation_loss_and_grad(x, tokens[:, None], torch.zeros(rows, 1, device=gpu_device))
    assert torch.all((loss + s.log_probs).abs() <= tol) and torch.all((grad + want[tokens]).abs() <= d_tol)
    leaf = x.contiguous().requires_grad_()
    back, = torch.autograd.grad(K.token_log_probs(leaf, tokens).log_probs.sum(), leaf)
    assert torch.all((back - want[tokens]).abs() <= d_tol)


def test_streams_and_graphs(K, gpu_device):
    """On a stream of its own and captured: the bits of the eager calls, replay after replay."""
    r = np.random.default_rng(11)
    x = on_gpu(crowd(r, 40, 50257), torch.float16, gpu_device, 0, 50304)
    t = torch.from_numpy(r.integers(0, 50257, size=40)).to(gpu_device)

    def step(logits):
        s = K.token_log_probs(logits, t, top=20)
        loss, grad = K.distillation_loss_and_grad(logits, s.top_tokens, s.top_log_probs, 2.0)
        leaf = logits.detach().requires_grad_()
        back, = torch.autograd.grad(K.token_log_probs(leaf, t).log_probs.sum(), leaf)
        return (*s, loss, grad, back)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(x)
    for seed in range(4):
        x.copy_(torch.from_numpy(crowd(np.random.default_rng(seed), 40, 50257)).half())
        graph.replay()
        want = step(x)
        for a, b in zip(captured, want):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
    assert len(other) == len(want)


def test_teacher_and_student(K, gpu_device):
    """The operators together: a GPT-2 teacher scores text, a student's last product learns from its top logits."""
    from gpt_triton_amd.gpt import FusedGPT, GPTConfig

    def model(width, seed):
        m = FusedGPT(GPTConfig(vocab_size=1003, block_size=64, n_layer=2, n_head=width // 64, n_embd=width, dropout=0.0))
        return m.init_synthetic_(seed, 0.08).half().to(gpu_device).eval()

    teacher, student = model(256, 1), model(128, 2)
    ids = torch.from_numpy(np.random.default_rng(12).integers(0, 1003, size=(4, 50))).to(gpu_device)
    with torch.no_grad():
        _, logits = teacher(ids, return_logits=True)
        hidden = student(ids)
    following = torch.full_like(ids, -100)
    following[:, :-1] = ids[:, 1:]
    s = K.token_log_probs(logits, following, top=16)
    x = host(logits).astype(np.float64).reshape(-1, 1003)
    z, _, lp, ent = want_scores(x, host(following).reshape(-1), 1.0)
    assert np.max(np.abs(host(s.log_probs).reshape(-1) - lp)) <= 2 * sum_error(1003) + 40 * U
    assert np.array_equal(host(s.top_tokens).reshape(-1, 16), top_ids(x, 16))
    assert torch.all(s.log_probs[:, -1] == 0)
    weights = (following >= 0).float()
    head = student.wte_weight.detach().float().requires_grad_()
    out = torch.matmul(hidden.float(), head.t())
    loss = K.distillation_loss(out, s.top_tokens, s.top_log_probs, 2.0, weights)
    loss.sum().backward()
    want, _, d, _ = want_distillation(host(out).astype(np.float64).reshape(-1, 1003), host(s.top_tokens).reshape(-1, 16),
                                      host(s.top_log_probs).reshape(-1, 16), 2.0, host(weights).reshape(-1))
    assert np.max(np.abs(host(loss).reshape(-1) - want)) <= 1e-5 * np.abs(want).max()
    d_head = d.T @ host(hidden).astype(np.float64).reshape(-1, 128)
    assert np.max(np.abs(host(head.grad) - d_head)) <= 1e-5 * np.abs(d_head).max()
