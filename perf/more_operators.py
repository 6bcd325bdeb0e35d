"""The operators of a training step that this framework has beside its losses, as cases that can be timed and compared:

  "attention"   flash_attention_packed in a training step: the output for whole prompts of different lengths, one behind
                the other without padding, and the gradients of q, k and v for the output's;
  "embeddings"  fused_embeddings in a training step: the rows of both tables, and the tables' gradients, dense;
  "clip"        clip_grad_norm_: the norm of all gradients of a model together, and the gradients, times a loss scale's
                inverse, at that norm or at the limit, in place or into tensors of their own.

`run` makes the framework's calls where `own` is set and computes the same in elementary torch operations
elsewhere.  `listed()` holds sizes that the benchmark, the configurations and the tests of this repository
name, and ordinary ones between and beyond them; `draw` gives more of the same ranges."""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "fp32": torch.float32}
# what the largest listed cases cost: attention's pairs times width and its plain form's scores, bytes of embeddings and
# gradients, elements of all gradients
MOST_PAIRS, MOST_SCORES = 1.7e11, 3.3e9
MOST_EMBEDDING_BYTES, MOST_GRADIENTS = 1.2e9, 3.6e8


def _attention(heads, kv_heads, d, lengths, fused):
    return {"op": "attention", "heads": heads, "kv_heads": kv_heads, "d": d,
            "lengths": " ".join(str(n) for n in lengths), "fused": fused}


def _embeddings(batch, seqlen, vocab, context, width, dtype):
    return {"op": "embeddings", "batch": batch, "seqlen": seqlen, "vocab": vocab, "context": context, "width": width,
            "dtype": dtype}


def _clip(layers, width, vocab, context, dtype, result, exceeded, loss_scale=1.0):
    return {"op": "clip", "layers": layers, "width": width, "vocab": vocab, "context": context, "dtype": dtype,
            "result": result, "exceeded": exceeded, "loss_scale": loss_scale}


def _ragged(rng, count, longest):
    """Lengths of `count` prompts of up to `longest` tokens: some of one token, one empty, the rest spread over
    the logarithm."""
    lengths = [int(math.exp(rng.uniform(0.0, math.log(longest + 0.999)))) for _ in range(count)]
    lengths[rng.randrange(count)] = longest
    if count > 4:
        lengths[rng.choice([i for i, n in enumerate(lengths) if n != longest] or [0])] = 0
    return lengths


def listed():
    rng = random.Random(23)
    cases = {
        # one short text of the 124M model: the smallest call
        "attention_1x24": _attention(12, 12, 64, [24], True),
        # a batch of documents of one token up to the context length, 124M
        "attention_48_ragged_1024": _attention(12, 12, 64, _ragged(rng, 48, 1024), True),
        # long texts, a key and value head for four query heads
        "attention_grouped_6x4096": _attention(32, 8, 128, [4096, 1933, 517, 4095, 64, 2049], False),
        # one very long text, 1600 wide
        "attention_1x8192": _attention(25, 25, 64, [8192], True),
        # two short texts in a model of some tests' size: latency
        "embeddings_2x70_small": _embeddings(2, 70, 512, 128, 256, "fp32"),
        # two texts of 124M: nearly all of the gradient is rows without a token
        "embeddings_2x64": _embeddings(2, 64, 50257, 1024, 768, "fp16"),
        # an ordinary training batch, fp32
        "embeddings_16x1024_fp32": _embeddings(16, 1024, 50304, 1024, 768, "fp32"),
        # the benchmark's batch
        "embeddings_512x300": _embeddings(512, 300, 50257, 1024, 768, "fp16"),
        # a small model's gradients, below the limit: latency
        "clip_small": _clip(2, 256, 512, 128, "fp32", "in place", False),
        # the 124M model's fp32 gradients on an ordinary step, below the limit
        "clip_124m_fp32": _clip(12, 768, 50304, 1024, "fp32", "in place", False),
        # fp16 gradients of a scaled loss, above the limit, into the optimizer's fp32 ones: the 1024-wide model
        "clip_medium_fp16_to_fp32": _clip(24, 1024, 50257, 1024, "fp16", "fp32", True, 1024.0),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_uniform(rng, low, high):
    return int(math.exp(rng.uniform(math.log(low), math.log(high + 0.999))))


def draw(rng):
    op = rng.choice(("attention", "attention", "embeddings", "clip"))
    if op == "attention":
        while True:
            heads, kv_heads = rng.choice(((12, 12), (16, 16), (25, 25), (32, 8), (32, 4), (16, 2), (8, 1)))
            d = rng.choice((16, 32, 64, 64, 64, 128, 128, 256))
            count, longest = _log_uniform(rng, 1, 64), _log_uniform(rng, 1, 8192)
            lengths = _ragged(rng, count, longest)
            if (sum(n * n for n in lengths) * heads * d <= MOST_PAIRS and sum(lengths) * heads * d <= 1 << 28 and
                    count * heads * longest * longest <= MOST_SCORES):
                return _attention(heads, kv_heads, d, lengths, rng.random() < 0.5)
    dtype = rng.choice(("fp16", "fp32"))
    if op == "embeddings":
        while True:
            vocab = rng.choice((50257, 50304, 32000, 65024, 128256, _log_uniform(rng, 300, 131072)))
            width = rng.choice((768, 768, 1024, 1280, 1600, _log_uniform(rng, 16, 2048)))
            seqlen = _log_uniform(rng, 1, 2048)
            case = _embeddings(_log_uniform(rng, 1, 1024), seqlen, vocab, seqlen + rng.choice((0, rng.randint(0, 1024))),
                               width, dtype)
            if work(case)["bytes"] <= MOST_EMBEDDING_BYTES:
                return case
    while True:
        width = rng.choice((256, 768, 1024, 1280, 1600, _log_uniform(rng, 16, 2048)))
        result = rng.choice(("in place", "fp32", "fp16"))
        exceeded = result != "in place" and rng.random() < 0.7
        case = _clip(_log_uniform(rng, 1, 48), width, rng.choice((50257, 50304, _log_uniform(rng, 300, 65536))),
                     rng.choice((512, 1024)), dtype, result, exceeded,
                     1.0 if result == "in place" or dtype == "fp32" else 1024.0)
        if sum(math.prod(shape) for shape in _shapes(case)) <= MOST_GRADIENTS:
            return case


def _lengths(case):
    return [int(n) for n in case["lengths"].split()]


def _shapes(case):
    """The parameters of a model, in the order that it has them."""
    h = case["width"]
    block = [(h,), (h,), (h, 3 * h), (3 * h,), (h, h), (h,), (h,), (h,), (h, 4 * h), (4 * h,), (4 * h, h), (h,)]
    return [(case["vocab"], h), (case["context"], h), *block * case["layers"], (h,), (h,)]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    state = {"op": case["op"]}
    if case["op"] == "attention":
        lengths = _lengths(case)
        n, g, d, total = case["heads"], case["kv_heads"], case["d"], sum(lengths)
        sizes = (n, g, g)
        if case["fused"]:  # q, k and v side by side in a row, as one product leaves them
            q, k, v = torch.randn(total, sum(sizes), d, generator=gen, device=dev, dtype=torch.float16).split(sizes, dim=1)
        else:
            q, k, v = (torch.randn(total, s, d, generator=gen, device=dev, dtype=torch.float16) for s in sizes)
        # what a scaled loss hands back, texts that count more and less among them
        d_out = torch.randn(total, n, d, generator=gen, device=dev, dtype=torch.float32)
        d_out *= torch.rand(total, 1, 1, generator=gen, device=dev) * 0.1
        starts = torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(dev)
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        # the lengths are a plain form's alone: it pads the sequences to the longest one
        return dict(state, q=q, k=k, v=v, d_out=d_out.half(), starts=starts, lengths=lengths)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "embeddings":
        vocab, h = case["vocab"], case["width"]
        # tokens of texts: the r-th most frequent one about 1 / r as often as the first
        rank = torch.rand(case["batch"], case["seqlen"], generator=gen, device=dev).mul_(math.log(vocab + 0.5)).exp_()
        ids = torch.randperm(vocab, generator=gen, device=dev)[rank.long().clamp_(max=vocab) - 1]
        wte = (torch.randn(vocab, h, generator=gen, device=dev) * 0.02).to(dtype).requires_grad_()
        wpe = (torch.randn(case["context"], h, generator=gen, device=dev) * 0.02).to(dtype).requires_grad_()
        d_out = (torch.randn(*ids.shape, h, generator=gen, device=dev) * 0.01).to(dtype)
        return dict(state, ids=ids, wte=wte, wpe=wpe, d_out=d_out)
    shapes = _shapes(case)
    sizes = [math.prod(shape) for shape in shapes]
    # the gradients of a model one behind the other in a buffer, as a data-parallel program keeps them
    spread = case["loss_scale"] * (3.0 if case["exceeded"] else 0.4) / math.sqrt(sum(sizes))
    flat = torch.randn(sum(sizes), generator=gen, device=dev, dtype=torch.float32).mul_(spread).to(dtype)

    def views(buffer):
        return [t.view(shape) for t, shape in zip(buffer.split(sizes), shapes)]

    result = flat if case["result"] == "in place" else torch.zeros_like(flat, dtype=DTYPES[case["result"]])
    return dict(state, grads=views(flat), out=None if result is flat else views(result), result=result, max_norm=1.0,
                scale=1.0 / case["loss_scale"])


# ---------------------------------------------------------------- plain forms
def _plain_attention(state):
    q, k, v, d_out, starts, lengths = (state[n].detach() if n in "qkv" else state[n] for n in
                                       ("q", "k", "v", "d_out", "starts", "lengths"))
    (total, n, d), g = q.shape, k.shape[1]
    count, longest, scale = len(lengths), max(lengths), 1.0 / math.sqrt(q.shape[2])
    row = torch.arange(longest, device=q.device)
    there = row < (starts[1:] - starts[:-1])[:, None]  # [count, longest]
    at = (starts[:-1, None] + row).clamp_(max=total - 1)

    def padded(t):  # [count * n, longest, d]
        t = t.float()[at] * there[..., None, None]
        return t.repeat_interleave(n // t.shape[2], dim=2).transpose(1, 2).reshape(count * n, longest, d)

    def packed(t, heads):  # [total, heads, d]
        t = t.view(count, heads, n // heads, longest, d).sum(dim=2).transpose(1, 2)
        return t[there].to(q.dtype)

    pq, pk, pv, pd = padded(q), padded(k), padded(v), padded(d_out)
    p = torch.bmm(pq * scale, pk.transpose(1, 2).contiguous())
    p.masked_fill_(row[None, :] > row[:, None], -math.inf)
    p -= p.amax(dim=2, keepdim=True)
    p.exp_()
    p /= p.sum(dim=2, keepdim=True)
    out = torch.bmm(p, pv)
    dv = torch.bmm(p.transpose(1, 2), pd)
    ds = torch.bmm(pd, pv.transpose(1, 2).contiguous())
    ds -= (pd * out).sum(dim=2, keepdim=True)
    ds *= p
    del p
    dq, dk = torch.bmm(ds, pk).mul_(scale), torch.bmm(ds.transpose(1, 2), pq).mul_(scale)
    return packed(out, n), packed(dq, n), packed(dk, g), packed(dv, g)


def _plain_embeddings(state):
    ids, wte, wpe, d_out = state["ids"], state["wte"].detach(), state["wpe"].detach(), state["d_out"]
    seqlen, h = ids.shape[1], wte.shape[1]
    out = (wte.float()[ids] + wpe.float()[:seqlen]).to(wte.dtype)
    d = d_out.float()
    d_wte = torch.zeros(wte.shape, device=d.device).index_add_(0, ids.view(-1), d.view(-1, h))
    d_wpe = torch.zeros(wpe.shape, device=d.device)
    d_wpe[:seqlen] = d.sum(dim=0)
    return out, d_wte.to(wte.dtype), d_wpe.to(wpe.dtype)


def _plain_clip(state):
    grads, out = state["grads"], state["out"] or state["grads"]
    norm = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt() * state["scale"]
    factor = state["scale"] * (state["max_norm"] / norm).clamp(max=1.0)
    [o.copy_(g.float() * factor) for g, o in zip(grads, out)]
    return norm, state["result"]


# ---------------------------------------------------------------- the framework's calls
def _own_attention(state):
    from gpt_triton_amd import kernels

    leaves = state["q"], state["k"], state["v"]
    out = kernels.flash_attention_packed(*leaves, state["starts"])
    return out, *torch.autograd.grad(out, leaves, state["d_out"])


def _own_embeddings(state):
    from gpt_triton_amd import kernels

    tables = state["wte"], state["wpe"]
    out = kernels.fused_embeddings(state["ids"], *tables)
    return out, *torch.autograd.grad(out, tables, state["d_out"])


def _own_clip(state):
    from gpt_triton_amd import kernels

    norm = kernels.clip_grad_norm_(state["grads"], state["max_norm"], scale=state["scale"], out=state["out"])
    return norm, state["result"]


_PLAIN = {"attention": _plain_attention, "embeddings": _plain_embeddings, "clip": _plain_clip}
_OWN = {"attention": _own_attention, "embeddings": _own_embeddings, "clip": _own_clip}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# ---------------------------------------------------------------- in 64 bits, from the definitions
def _exact_attention(state):
    q, k, v, d_out = (state[name].detach() for name in ("q", "k", "v", "d_out"))
    (total, n, d), g = q.shape, k.shape[1]
    out, dq = (torch.empty(total, n, d, dtype=torch.float64, device=q.device) for _ in range(2))
    dk, dv = (torch.zeros(total, g, d, dtype=torch.float64, device=q.device) for _ in range(2))
    first = 0
    for length in state["lengths"]:
        at = slice(first, first + length)
        first += length
        past = torch.ones(length, length, dtype=torch.bool, device=q.device).tril_()
        for h in range(n):
            a, b, c, e = q[at, h].double(), k[at, h * g // n].double(), v[at, h * g // n].double(), d_out[at, h].double()
            w = torch.softmax(torch.where(past, a @ b.T * d ** -0.5, -math.inf), dim=1)
            out[at, h] = w @ c
            dv[at, h * g // n] += w.T @ e
            dw = e @ c.T
            ds = w * (dw - (w * dw).sum(dim=1, keepdim=True)) * d ** -0.5
            dq[at, h] = ds @ b
            dk[at, h * g // n] += ds.T @ a
    return out, dq, dk, dv


def _exact_embeddings(state):
    ids, wte, wpe, d = state["ids"].view(-1), state["wte"].detach(), state["wpe"].detach(), state["d_out"].double()
    batch, seqlen, h = d.shape
    place = torch.arange(seqlen, device=d.device).repeat(batch)
    out = (wte.double().index_select(0, ids) + wpe.double().index_select(0, place)).view(d.shape)
    # sums of each token's rows: differences of the running sum over the rows in the order of their tokens
    order = torch.argsort(ids)
    d_wte = torch.zeros(wte.shape, dtype=torch.float64, device=d.device)
    tokens, counts = torch.unique_consecutive(ids[order], return_counts=True)
    ends = counts.cumsum(0)
    for first in range(0, h, 256):
        columns = slice(first, min(first + 256, h))
        running = d.view(-1, h)[:, columns][order].cumsum(0)
        sums = running[ends - 1]
        sums[1:] -= running[ends[:-1] - 1]
        d_wte[tokens, columns] = sums
    d_wpe = torch.zeros(wpe.shape, dtype=torch.float64, device=d.device)
    for text in d:
        d_wpe[:seqlen] += text
    return out, d_wte, d_wpe


def _exact_clip(state):
    norm = math.sqrt(sum(float(torch.linalg.vector_norm(g, dtype=torch.float64)) ** 2 for g in state["grads"]))
    norm *= state["scale"]
    factor = state["scale"] * min(1.0, state["max_norm"] / norm)
    flat = torch.cat([g.reshape(-1) for g in state["grads"]]).double()
    return torch.tensor(norm, dtype=torch.float64), flat.mul_(factor)


_EXACT = {"attention": _exact_attention, "embeddings": _exact_embeddings, "clip": _exact_clip}


def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed))


def work(case):
    if case["op"] == "attention":
        lengths = _lengths(case)
        n, g, d, total = case["heads"], case["kv_heads"], case["d"], sum(lengths)
        # q, k, v and the output's gradient read, the output and the three gradients written; two products forward, and
        # backward four, and the scores once more
        return {"bytes": 2 * d * total * (4 * n + 4 * g) + 8 * (len(lengths) + 1),
                "flops": 14 * n * d * sum(m * (m + 1) // 2 for m in lengths)}
    size = 2 if case["dtype"] == "fp16" else 4
    if case["op"] == "embeddings":
        rows, h = case["batch"] * case["seqlen"], case["width"]
        # rows of the token table that a batch reads: no more than there are
        read = min(rows, case["vocab"]) + case["seqlen"]
        return {"bytes": size * h * (read + 2 * rows + case["vocab"] + case["context"]) + 8 * rows, "flops": 3 * rows * h}
    elements = sum(math.prod(shape) for shape in _shapes(case))
    written = 0 if case["result"] == "in place" and not case["exceeded"] else 2 if case["result"] == "fp16" else 4
    return {"bytes": elements * (size + written), "flops": 2 * elements + (elements if written else 0)}
