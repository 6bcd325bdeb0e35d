"""A student's training step out of the operators that have gradients, torch's products between them: embeddings, attention over
packed texts, the loss against a teacher's top logits, all gradients clipped together.  Against the same step with the
operators' formulas in torch, whose numbers are rounded to fp16 in the same places but inside attention.

There the forward and the backward pass round some 6 numbers of a chain to fp16 (weights, u, delta's output, and each result),
2^-11 of themselves at most, and what they change is rounded anew in each of the 4 fp16 results behind: 2-norms of gradients
may differ by 2^-11 times the square root of 6 + 2 * 4 in typical cases, and by 14 * 2^-11 at most, to the first order."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

V, P, H, N, G, D = 400, 96, 128, 4, 2, 32
LENGTHS = [64, 1, 30, 0, 95]


def parameters(device):
    r = torch.Generator().manual_seed(0)
    new = lambda *shape, by=0.2: (torch.randn(*shape, generator=r) * by).to(device).requires_grad_()
    return [new(V, H), new(P, H), new(H, (N + 2 * G) * D), new(N * D, H)]


def attention(q, k, v, lengths):
    """In fp32, rounded once."""
    out, first = [], 0
    for length in lengths:
        a, b, c = (t[first:first + length].float().transpose(0, 1) for t in (q, k, v))
        first += length
        b, c = (t.repeat_interleave(N // G, 0) for t in (b, c))
        s = (a @ b.transpose(1, 2).contiguous()) * D ** -0.5
        past = torch.ones(length, length, dtype=torch.bool, device=q.device).tril_()
        out.append((torch.softmax(s.masked_fill(~past, -math.inf), 2) @ c).transpose(0, 1))
    return torch.cat(out).half()


def distillation(logits, ids, values):
    log_q = torch.log_softmax(values, 1)
    return (log_q.exp() * (log_q - torch.log_softmax(logits.float(), 1).gather(1, ids))).sum(1)


def step(K, params, batch, own):
    wte, wpe, w_qkv, w_out = params
    tokens, rows, starts, ids, values = batch
    if own:
        x = K.fused_embeddings(tokens, wte, wpe)
    else:
        x = wte[tokens] + wpe[:tokens.shape[1]]
    x = x.view(-1, H)[rows]  # the texts without their padding
    q, k, v = (x @ w_qkv).half().view(-1, N + 2 * G, D).split((N, G, G), dim=1)
    y = K.flash_attention_packed(q, k, v, starts) if own else attention(q, k, v, LENGTHS)
    x = x + y.reshape(-1, N * D).float() @ w_out
    logits = x @ wte.t()
    losses = K.distillation_loss(logits, ids, values) if own else distillation(logits, ids, values)
    return losses, torch.autograd.grad(losses.sum() * 8.0, params)  # a loss scale


def batch_of(device, seed):
    r = np.random.default_rng(seed)
    to = lambda t: torch.from_numpy(t).to(device)
    tokens = to(r.integers(0, V, (len(LENGTHS), P)))
    rows = to(np.concatenate([s * P + np.arange(n) for s, n in enumerate(LENGTHS)]))
    starts = to(np.concatenate(([0], np.cumsum(LENGTHS))))
    ids = to(np.stack([r.permutation(V)[:8] for _ in range(sum(LENGTHS))]))
    return tokens, rows, starts, ids, to((r.standard_normal((sum(LENGTHS), 8)) * 2).astype(np.float32))


def test_step(gpu_device):
    from gpt_triton_amd import kernels as K

    params, batch = parameters(gpu_device), batch_of(gpu_device, 1)
    losses, grads = step(K, params, batch, True)
    want_losses, want = step(K, params, batch, False)
    assert float((losses - want_losses).detach().norm()) <= 14 * 2.0**-11 * float(want_losses.detach().norm())
    for g, w in zip(grads, want):
        assert float((g - w).norm()) <= 14 * 2.0**-11 * float(w.norm())
    norm = math.sqrt(sum(float(g.double().pow(2).sum()) for g in grads)) / 8
    kept = [g.clone() for g in grads]
    got = K.clip_grad_norm_(grads, norm / 3, scale=1 / 8)
    assert abs(float(got) - norm) <= 2.0**-22 * norm
    for g, w in zip(grads, kept):
        assert torch.all((g - w / 24).abs() <= 2.0**-21 * (w / 24).abs())


def test_captured_step(gpu_device):
    """Replayed for new texts and parameters, with the program's eager steps between."""
    from gpt_triton_amd import kernels as K

    params, batch = parameters(gpu_device), batch_of(gpu_device, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.clip_grad_norm_(step(K, params, batch, True)[1], 1.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        losses, grads = step(K, params, batch, True)
        norm = K.clip_grad_norm_(grads, 0.5)
    for seed in (3, 4, 5):
        for old, new in zip(batch, batch_of(gpu_device, seed)):
            old.copy_(new)
        with torch.no_grad():
            for p in params:
                p.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        eager_losses, eager = step(K, [p.detach().clone().requires_grad_() for p in params], batch, True)
        eager_norm = K.clip_grad_norm_(eager, 0.5)
        # torch's products may take other kernels under capture
        assert float((losses - eager_losses).detach().norm()) <= 2.0**-9 * float(eager_losses.detach().norm())
        assert abs(float(norm) - float(eager_norm)) <= 2.0**-9 * float(eager_norm)
        for g, w in zip(grads, eager):
            assert float((g - w).norm()) <= 2.0**-9 * float(w.norm())
