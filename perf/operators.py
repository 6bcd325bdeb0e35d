"""The operators for scoring texts and learning from the scores, as cases that can be timed and compared:

  "attention"  flash_attention_packed: causal attention over whole prompts of different lengths, one behind
               the other without padding, grouped heads;
  "scores"     token_log_probs: the log probability of a given token in each row of logits, the row's entropy
               and its most likely tokens; with "train" the gradient of the logits too;
  "distil"     distillation_loss (the losses; with "train" "autograd" a backward pass behind it) and
               distillation_loss_and_grad ("train" "one pass"): a teacher's top logits against a student's.

`run` makes the framework's calls where `own` is set and computes the same in elementary torch operations
elsewhere.  `listed()` holds sizes that the benchmark, the configurations and the tests of this repository
name, and ordinary ones between and beyond them; `draw` gives more of the same ranges."""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "fp32": torch.float32}
LONGEST = 16384


def _attention(heads, kv_heads, d, lengths, fused):
    return {"op": "attention", "heads": heads, "kv_heads": kv_heads, "d": d,
            "lengths": " ".join(str(n) for n in lengths), "fused": fused}


def _scores(rows, vocab, dtype, padded, top, temperature=1.0, masked=False, train=False):
    return {"op": "scores", "rows": rows, "vocab": vocab, "dtype": dtype, "padded": padded, "top": top,
            "temperature": temperature, "masked": masked, "train": train}


def _distil(rows, vocab, dtype, padded, top, temperature, train):
    return {"op": "distil", "rows": rows, "vocab": vocab, "dtype": dtype, "padded": padded, "top": top,
            "temperature": temperature, "train": train}


def _ragged(rng, count, longest):
    """Lengths of `count` prompts of up to `longest` tokens: some of one token, one empty, the rest spread over
    the logarithm."""
    lengths = [int(math.exp(rng.uniform(0.0, math.log(longest + 0.999)))) for _ in range(count)]
    lengths[rng.randrange(count)] = longest
    if count > 4:
        lengths[rng.choice([i for i, n in enumerate(lengths) if n != longest] or [0])] = 0
    return lengths


def listed():
    rng = random.Random(20)
    cases = {
        # one short prompt of the 124M model, the q, k, v product's output as it is: the smallest call
        "attention_1x24": _attention(12, 12, 64, [24], True),
        # documents of one token up to the context length, scored together by the 124M model
        "attention_48_ragged_1024": _attention(12, 12, 64, _ragged(rng, 48, 1024), True),
        # long prompts of a model with a key and value head for four query heads
        "attention_grouped_6x4096": _attention(32, 8, 128, [4096, 1933, 517, 4095, 64, 2049], False),
        # one very long prompt, 1600 wide
        "attention_1x16384": _attention(25, 25, 64, [LONGEST], True),
        # the next token's alternatives of one prompt, rows as the LM head pads them: latency
        "scores_1_top20": _scores(1, 50257, "fp16", True, 20),
        # a text's log likelihood, from the LM head's padded rows
        "scores_1477": _scores(1477, 50257, "fp16", True, 0),
        # texts with alternatives for each token, dense rows of odd length, a vocabulary cut by a mask
        "scores_4096_top5_odd": _scores(4096, 50257, "fp16", False, 5, 0.8, masked=True),
        # log probabilities and entropy in a training step, fp32 logits
        "scores_train_2048_fp32": _scores(2048, 50304, "fp32", False, 0, train=True),
        # a few rows compared with their teacher
        "distil_24": _distil(24, 50257, "fp16", True, 20, 1.0, "none"),
        # an ordinary step of a student
        "distil_2048": _distil(2048, 50257, "fp16", True, 64, 2.0, "one pass"),
        # the same in fp32, as many top logits as are taken
        "distil_4096_fp32": _distil(4096, 50304, "fp32", False, 128, 1.0, "one pass"),
        # a large batch whose loss torch's own graph goes on from
        "distil_16384_autograd": _distil(16384, 50304, "fp16", False, 32, 1.0, "autograd"),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_uniform(rng, low, high):
    return int(math.exp(rng.uniform(math.log(low), math.log(high + 0.999))))


def draw(rng):
    op = rng.choice(("attention", "scores", "distil"))
    if op == "attention":
        while True:
            heads, kv_heads = rng.choice(((12, 12), (16, 16), (25, 25), (32, 8), (32, 4), (16, 2), (8, 1)))
            d = rng.choice((16, 32, 64, 64, 64, 128, 128, 256))
            count, longest = _log_uniform(rng, 1, 64), _log_uniform(rng, 1, LONGEST)
            lengths = _ragged(rng, count, longest)
            # as much work as the largest listed case, and scores that a plain form has room for
            if (sum(n * n for n in lengths) * heads * d <= LONGEST * LONGEST * 25 * 64 and
                    count * heads * longest * longest <= LONGEST * LONGEST * 25 and
                    sum(lengths) * heads * d <= 1 << 28):
                return _attention(heads, kv_heads, d, lengths, rng.random() < 0.5)
    vocab = rng.choice((50257, 50304, 32000, 65024, 128256, _log_uniform(rng, 300, 131072)))
    dtype = rng.choice(("fp16", "fp16", "fp32"))
    padded = rng.random() < 0.5
    most = 16384 * 50304 * 2 // (vocab * (2 if dtype == "fp16" else 4))
    temperature = rng.choice((1.0, 1.0, 0.7, 2.0))
    if op == "scores":
        train = rng.random() < 0.3
        rows = _log_uniform(rng, 1, min(most // 2, 8192 if train else 4096))
        top = 0 if train else rng.choice((0, 1, 5, 20, rng.randint(2, 128)))
        return _scores(rows, vocab, dtype, padded, top, temperature, not train and rng.random() < 0.3, train)
    rows = _log_uniform(rng, 1, min(most, 16384))
    return _distil(rows, vocab, dtype, padded, rng.choice((8, 20, 64, rng.randint(1, 128))), temperature,
                   rng.choice(("none", "one pass", "one pass", "autograd")))


def _lengths(case):
    return [int(n) for n in case["lengths"].split()]


def _logits(case, gen, dev):
    """Logits of trained models' kind: a broad crowd and in each row a few tokens far above it.  [rows, vocab],
    dense or the front of rows that are padded to a multiple of 64 with zeros, as the LM head leaves them."""
    rows, vocab = case["rows"], case["vocab"]
    width = -(-vocab // 64) * 64 if case["padded"] else vocab
    x = torch.randn(rows, width, generator=gen, device=dev, dtype=torch.float32).mul_(2.2).sub_(3.0)
    # one in each sixth of the vocabulary: different tokens, since a scatter to the same place twice keeps either
    sixth = vocab // 6
    liked = torch.randint(0, sixth, (rows, 6), generator=gen, device=dev) + torch.arange(6, device=dev) * sixth
    x.scatter_(1, liked, torch.rand(rows, 6, generator=gen, device=dev) * 16.0)
    x[:, vocab:] = 0.0
    return x.to(DTYPES[case["dtype"]])[:, :vocab], liked


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    state = {"op": case["op"]}
    if case["op"] == "attention":
        lengths = _lengths(case)
        n, g, d, total = case["heads"], case["kv_heads"], case["d"], sum(lengths)
        sizes = (n, g, g)
        if case["fused"]:  # q, k and v side by side in a row, as one product leaves them
            y = torch.randn(total, sum(sizes), d, generator=gen, device=dev, dtype=torch.float16)
            q, k, v = y.split(sizes, dim=1)
        else:
            q, k, v = (torch.randn(total, s, d, generator=gen, device=dev, dtype=torch.float16) for s in sizes)
        starts = torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(dev)
        # the lengths are a plain form's alone: it pads the sequences to the longest one
        return dict(state, q=q, k=k, v=v, starts=starts, lengths=lengths)
    rows, vocab = case["rows"], case["vocab"]
    logits, liked = _logits(case, gen, dev)
    state["temperature"] = case["temperature"]
    if case["op"] == "scores":
        # half of the tokens are ones that the model likes
        tokens = torch.randint(0, vocab, (rows,), generator=gen, device=dev)
        tokens = torch.where(torch.rand(rows, generator=gen, device=dev) < 0.5, liked[:, 0], tokens)
        if case["masked"]:  # a fifth of the vocabulary is not allowed, the given tokens are
            hidden = torch.rand(vocab, generator=gen, device=dev) < 0.2
            kept = logits.gather(1, tokens[:, None])
            logits.masked_fill_(hidden, -math.inf)
            logits.scatter_(1, tokens[:, None], kept)
        state.update(tokens=tokens, top=case["top"], train=case["train"])
        if case["train"]:
            # what the rest of a loss hands back: a weight for each token, a bonus for entropy
            state["d_log_probs"] = -torch.rand(rows, generator=gen, device=dev)
            state["d_entropy"] = torch.full((rows,), -0.01, device=dev)
            logits.requires_grad_()
        return dict(state, logits=logits)
    # a teacher that agrees with the student in part: its top logits fall off with the rank
    k = case["top"]
    ids = torch.rand(rows, vocab, generator=gen, device=dev).topk(k, dim=1).indices if vocab <= 4096 else (
        torch.randint(0, vocab // k, (rows, k), generator=gen, device=dev) +
        torch.arange(k, device=dev) * (vocab // k))
    values = torch.randn(rows, k, generator=gen, device=dev) * 3.0
    state.update(ids=ids, values=values, train=case["train"],
                 # a loss scale's share for each row; an eighth of the rows is padding
                 weights=torch.where(torch.rand(rows, generator=gen, device=dev) < 0.125, 0.0, 64.0))
    if case["train"] == "autograd":
        logits.requires_grad_()
    return dict(state, logits=logits)


# ---------------------------------------------------------------- plain forms
def _plain_attention(state):
    q, k, v, starts, lengths = (state[n] for n in ("q", "k", "v", "starts", "lengths"))
    (total, n, d), g = q.shape, k.shape[1]
    count, longest = len(lengths), max(lengths)
    row = torch.arange(longest, device=q.device)
    there = row < (starts[1:] - starts[:-1])[:, None]  # [count, longest]
    at = (starts[:-1, None] + row).clamp_(max=total - 1)

    def padded(t):  # [count * n, longest, d]
        t = t.float()[at] * there[..., None, None]
        return t.repeat_interleave(n // t.shape[2], dim=2).transpose(1, 2).reshape(count * n, longest, d)

    keys = padded(k).transpose(1, 2).contiguous()
    s = torch.bmm(padded(q) / math.sqrt(d), keys)
    s.masked_fill_(row[None, :] > row[:, None], -math.inf)
    s -= s.amax(dim=2, keepdim=True)
    s.exp_()
    s /= s.sum(dim=2, keepdim=True)
    out = torch.bmm(s, padded(v)).view(count, n, longest, d).transpose(1, 2)
    return out[there].to(q.dtype)


def _normalised(logits, temperature):
    """(log softmax of the scaled logits, its exponentials), fp32."""
    z = logits.detach().float()
    if temperature != 1.0:
        z = z / temperature
    z = z - z.amax(dim=1, keepdim=True)
    p = z.exp()
    total = p.sum(dim=1, keepdim=True)
    return z.sub_(total.log()), p.div_(total)


def _plain_scores(state):
    logits, tokens, top = state["logits"], state["tokens"], state["top"]
    z, p = _normalised(logits, state["temperature"])
    log_probs = z.gather(1, tokens[:, None])[:, 0]
    terms = (p * z).masked_fill_(p == 0, 0.0)  # 0 log 0
    entropy = -terms.sum(dim=1)
    if state["train"]:
        g, h = state["d_log_probs"][:, None], state["d_entropy"][:, None]
        d = -(p * g) - h * (terms + p * entropy[:, None])
        d.scatter_add_(1, tokens[:, None], g)
        return log_probs, entropy, (d / state["temperature"]).to(logits.dtype)
    if top == 0:
        return log_probs, entropy
    # equal logits in the order of their ids: a stable sort
    ids = torch.sort(logits.detach(), dim=1, descending=True, stable=True).indices[:, :top]
    return log_probs, entropy, z.gather(1, ids), ids


def _plain_distil(state):
    logits, ids, tau, w = state["logits"], state["ids"], state["temperature"], state["weights"]
    z, p = _normalised(logits, tau)
    log_q = state["values"] / tau
    log_q = log_q - log_q.amax(dim=1, keepdim=True)
    log_q = log_q - log_q.exp().sum(dim=1, keepdim=True).log()
    q = log_q.exp()
    losses = w * (q * (log_q - z.gather(1, ids))).sum(dim=1)
    if state["train"] == "none":
        return losses
    d = p.scatter_add_(1, ids, -q).mul_((w / tau)[:, None])
    return losses, d.to(logits.dtype)


# ---------------------------------------------------------------- the framework's calls
def _own_attention(state):
    from gpt_triton_amd import kernels

    return kernels.flash_attention_packed(state["q"], state["k"], state["v"], state["starts"])


def _own_scores(state):
    from gpt_triton_amd import kernels

    logits, top = state["logits"], state["top"]
    r = kernels.token_log_probs(logits, state["tokens"], top=top, temperature=state["temperature"])
    if state["train"]:
        grad, = torch.autograd.grad((r.log_probs, r.entropy), logits, (state["d_log_probs"], state["d_entropy"]))
        return r.log_probs, r.entropy, grad
    return (r.log_probs, r.entropy, r.top_log_probs, r.top_tokens) if top else (r.log_probs, r.entropy)


def _own_distil(state):
    from gpt_triton_amd import kernels

    logits = state["logits"]
    rest = state["ids"], state["values"], state["temperature"], state["weights"]
    if state["train"] == "one pass":
        return kernels.distillation_loss_and_grad(logits, *rest)
    losses = kernels.distillation_loss(logits, *rest)
    if state["train"] == "none":
        return losses
    grad, = torch.autograd.grad(losses.sum(), logits)
    return losses, grad


_PLAIN = {"attention": _plain_attention, "scores": _plain_scores, "distil": _plain_distil}
_OWN = {"attention": _own_attention, "scores": _own_scores, "distil": _own_distil}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# ---------------------------------------------------------------- in 64 bits, from the definitions
def _exact_attention(state):
    q, k, v = state["q"], state["k"], state["v"]
    (total, n, d), g = q.shape, k.shape[1]
    out = torch.empty(total, n, d, dtype=torch.float64, device=q.device)
    first = 0
    for length in state["lengths"]:
        at = slice(first, first + length)
        first += length
        past = torch.ones(length, length, dtype=torch.bool, device=q.device).tril_()
        for h in range(n):
            a, b, c = q[at, h].double(), k[at, h * g // n].double(), v[at, h * g // n].double()
            w = torch.where(past, a @ b.T * d ** -0.5, -math.inf)
            out[at, h] = torch.softmax(w, dim=1) @ c
    return out


def _exact_rows(state, rows):
    """What `run` returns of these rows but for the top tokens, which are whole numbers."""
    x = state["logits"].detach()[rows].double() / state["temperature"]
    z = torch.log_softmax(x, dim=1)
    p = torch.exp(z)
    if state["op"] == "distil":
        ids, w = state["ids"][rows], state["weights"][rows].double()
        log_q = torch.log_softmax(state["values"][rows].double() / state["temperature"], dim=1)
        q = torch.exp(log_q)
        losses = w * (q * (log_q - z.gather(1, ids))).sum(1)
        if state["train"] == "none":
            return [losses]
        target = torch.zeros_like(p).scatter_add_(1, ids, q)
        return [losses, (p - target) * w[:, None] / state["temperature"]]
    tokens = state["tokens"][rows]
    log_p = z.gather(1, tokens[:, None]).squeeze(1)
    entropy = torch.special.entr(p).sum(1)
    if state["train"]:
        g, h = state["d_log_probs"][rows].double()[:, None], state["d_entropy"][rows].double()[:, None]
        one = torch.zeros_like(p).scatter_(1, tokens[:, None], 1.0)
        d = g * (one - p) + h * (torch.special.entr(p) - p * entropy[:, None])
        return [log_p, entropy, d / state["temperature"]]
    if state["top"] == 0:
        return [log_p, entropy]
    return [log_p, entropy, torch.topk(z, state["top"], dim=1).values]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(state)
    parts = [_exact_rows(state, slice(r, r + 512)) for r in range(0, case["rows"], 512)]
    out = [torch.cat(p) for p in zip(*parts)]
    if case["op"] == "scores" and case["top"]:
        out.append(None)
    return out if len(out) > 1 else out[0]


def work(case):
    if case["op"] == "attention":
        lengths = _lengths(case)
        n, g, d = case["heads"], case["kv_heads"], case["d"]
        return {"bytes": 2 * d * (2 * n + 2 * g) * sum(lengths) + 8 * (len(lengths) + 1),
                "flops": 4 * n * d * sum(m * (m + 1) // 2 for m in lengths)}
    size = 2 if case["dtype"] == "fp16" else 4
    rows, matrix = case["rows"], case["rows"] * case["vocab"]
    train = case["train"] not in (False, "none")
    if case["op"] == "scores":
        rest = rows * (8 + 4 + 4 + 12 * case["top"] + (8 if train else 0))
    else:
        rest = rows * (12 * case["top"] + 4 + 4)
    return {"bytes": matrix * size * (2 if train else 1) + rest, "flops": matrix * (8 if train else 4)}
