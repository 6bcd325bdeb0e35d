"""flash_attention_packed against its formula in 64 bits.

Tolerance, from the arithmetic (u = 2^-24, half a step of fp32; h = 2^-11, half a step of fp16):
  * a score is a sum of d products in fp32: off by (d + 8) u times the sum of their sizes, times the scale.  Its exponent is
    rounded twice more, relative to itself and to the row's maximum.  Both move a weight by E relative, E the
    largest such error of the row in natural units, and the hardware's exponential by 2 u;
  * a weight is rounded to fp16 for the product with v, relative to the row's largest weight: h of itself, or 2^-25 where
    it is a subnormal number, while the denominator sums L of them in fp32;
  * an output is rounded to fp16: h of itself, at least 2^-25.
With A = sum w |v|: |error| <= (h + 2 E + 8 u + L u) A + L 2^-25 max |v| + h |out| + 2^-25."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U, H = 2.0**-24, 2.0**-11


@pytest.fixture(scope="module")
def K(gpu_device):
    from gpt_triton_amd import kernels

    return kernels


def want(q, k, v, scale):
    """(out, tolerance) of one sequence, [L, N, d] fp16 tensors, in 64 bits."""
    L, n, d = q.shape
    rep = n // k.shape[1]
    out, tol = torch.empty(L, n, d, dtype=torch.float64, device=q.device), torch.empty(L, n, d, dtype=torch.float64,
                                                                                       device=q.device)
    past = torch.ones(L, L, dtype=torch.bool, device=q.device).tril_()
    for i in range(n):
        a, b, c = q[:, i].double(), k[:, i // rep].double(), v[:, i // rep].double()
        s = torch.where(past, torch.mm(a, b.t().contiguous()) * scale, -math.inf)
        w = torch.softmax(s, 1)
        size = torch.where(past, torch.mm(a.abs(), b.abs().t().contiguous()) * scale, 0.0).amax(1, keepdim=True)
        e = (d + 16) * U * size
        out[:, i] = torch.mm(w, c)
        A = torch.mm(w, c.abs())
        tol[:, i] = ((H + 2 * e + (8 + L) * U) * A + L * 2.0**-25 * c.abs().amax() + H * out[:, i].abs() + 2.0**-25)
    return out, tol


def make(r, total, n, g, d, fused, device, spread=1.0):
    sizes = (n, g, g)
    if fused:
        y = torch.from_numpy((r.standard_normal((total, sum(sizes), d)) * spread).astype(np.float16)).to(device)
        return y.split(sizes, dim=1)
    return tuple(torch.from_numpy((r.standard_normal((total, s, d)) * spread).astype(np.float16)).to(device) for s in sizes)


def starts_of(lengths, device, first=0):
    return torch.tensor([first] + [first + int(x) for x in np.cumsum(lengths)], dtype=torch.int64, device=device)


def check(K, q, k, v, lengths, scale=None, first=0):
    out = K.flash_attention_packed(q, k, v, starts_of(lengths, q.device, first), scale=scale)
    assert out.shape == q.shape and out.is_contiguous()
    at = first
    for L in lengths:
        rows = slice(at, at + L)
        at += L
        if L:
            w, tol = want(q[rows], k[rows], v[rows], q.shape[2] ** -0.5 if scale is None else scale)
            err = (out[rows].double() - w).abs()
            assert torch.all(err <= tol), (L, float((err / tol).max()))
    return out


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
@pytest.mark.parametrize("heads", [(1, 1), (7, 7), (8, 8), (9, 9), (32, 8), (6, 1), (36, 9), (64, 16)])
def test_heads(K, gpu_device, d, heads):
    r = np.random.default_rng(heads[0])
    lengths = [150, 64, 3, 97]
    check(K, *make(r, sum(lengths), *heads, d, True, gpu_device), lengths)


@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
def test_many_blocks(K, gpu_device, d):
    """More blocks than run at once: 32 queries a wavefront, the heaviest blocks first (few sequences, few blocks) or in
    the order of the slots (more than 256 sequences, or hardly a block each), with and without heads that one XCD has."""
    r = np.random.default_rng(19)
    for heads, lengths in (((64, 16), [700, 33, 0, 512, 255, 1]), ((20, 20), [65, 1000, 129, 0, 640, 2000]),
                           ((48, 12), r.integers(0, 30, 300).tolist()), ((72, 9), [1500, 31, 900, 2100]), ((64, 64), [1600]),
                           ((64, 8), [1] * 200 + [100, 200])):
        q, k, v = make(r, sum(lengths), *heads, d, True, gpu_device)
        out = K.flash_attention_packed(q, k, v, starts_of(lengths, gpu_device))
        ends = np.cumsum(lengths)
        for s in {0, 1, len(lengths) // 2, len(lengths) - 1, int(np.argmax(lengths))} & set(range(len(lengths))):
            rows = slice(int(ends[s]) - lengths[s], int(ends[s]))
            some = [0, heads[0] // 2, heads[0] - 1]
            rep = heads[0] // heads[1]
            for h in some:
                if lengths[s]:
                    w, tol = want(q[rows, h:h + 1], k[rows, h // rep:h // rep + 1], v[rows, h // rep:h // rep + 1], d ** -0.5)
                    assert torch.all((out[rows, h:h + 1].double() - w).abs() <= tol), (heads, s, h)
        assert torch.all(torch.isfinite(out))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", [(72, 9), (80, 16)])
def test_long_in_the_order_of_slots(K, gpu_device, d, heads):
    """Too many blocks for the heaviest of all heads to come first."""
    lengths = [3000, 5100, 0, 2500]
    q, k, v = make(np.random.default_rng(27), sum(lengths), *heads, d, True, gpu_device)
    out = K.flash_attention_packed(q, k, v, starts_of(lengths, gpu_device))
    rep = heads[0] // heads[1]
    for first, L in ((0, 3000), (8100, 2500)):
        rows = slice(first, first + L)
        for h in (0, 35, heads[0] - 1):
            w, tol = want(q[rows, h:h + 1], k[rows, h // rep:h // rep + 1], v[rows, h // rep:h // rep + 1], d ** -0.5)
            assert torch.all((out[rows, h:h + 1].double() - w).abs() <= tol), (L, h)
    assert torch.all(torch.isfinite(out))


@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("heads", [12, 25, 40, 64])
@pytest.mark.parametrize("lengths", [[191, 320, 640, 7], [1000, 1, 383], [64, 128, 1024, 192]])
def test_every_deal(K, gpu_device, d, heads, lengths):
    """By the number of heads: 16 and 32 queries a wavefront with the key tiles in two parts, 16 and 32 in one."""
    q, k, v = make(np.random.default_rng(26), sum(lengths), heads, heads, d, True, gpu_device)
    out = K.flash_attention_packed(q, k, v, starts_of(lengths, gpu_device))
    ends = np.cumsum(lengths)
    for end, L in zip(ends, lengths):
        rows = slice(int(end) - L, int(end))
        for h in (0, heads // 2, heads - 1):
            w, tol = want(q[rows, h:h + 1], k[rows, h:h + 1], v[rows, h:h + 1], d ** -0.5)
            assert torch.all((out[rows, h:h + 1].double() - w).abs() <= tol), (L, h)
    assert torch.all(torch.isfinite(out))


@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
def test_long(K, gpu_device, d):
    r = np.random.default_rng(7)
    lengths = [3001, 5, 1500]
    check(K, *make(r, sum(lengths), 2, 1, d, True, gpu_device), lengths)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale,spread", [(0.02, 1.0), (1.0, 1.0), (0.125, 6.0), (0.125, 0.01)])
def test_sharp_and_flat_weights(K, gpu_device, d, scale, spread):
    """Scores of up to some hundred, where a weight or two are left of a row, and ones that are all alike."""
    r = np.random.default_rng(8)
    lengths = [700, 33]
    check(K, *make(r, sum(lengths), 2, 2, d, False, gpu_device, spread), lengths, scale=scale)


@pytest.mark.parametrize("d", [64, 128])
def test_scores_that_rise_and_fall(K, gpu_device, d):
    """The running maximum moves in every tile, or never after the first; and leaps by more than weights reach."""
    r = np.random.default_rng(9)
    L = 900
    q, k, v = make(r, L, 2, 2, d, False, gpu_device)
    q[:] = 0
    q[:, :, 0] = 1.0
    ramp = torch.arange(L, device=gpu_device)
    for values in (ramp * 0.25, -ramp * 0.25, (ramp // 100) * 40.0, (ramp % 130) * 1.0, 200.0 - (ramp // 64) * 14.0):
        k[:, :, 0] = values[:, None].half()
        check(K, q, k, v, [L], scale=1.0)


@pytest.mark.parametrize("d", [16, 64, 128, 256])
def test_scores_beyond_the_exponent(K, gpu_device, d):
    """Scores so large that fp32 exponents are off by more than weights reach, and the largest fp16 inputs."""
    r = np.random.default_rng(20)
    L = 200
    q, k, v = make(r, L, 2, 2, d, False, gpu_device)
    for scale, size in ((1e4, 100.0), (1e15, 1.0), (1.0, 65504.0), (1e-20, 1.0)):
        a, b = (q.sign() * size, k.sign() * size) if size > 1e3 else (q * size, k * size)
        out = K.flash_attention_packed(a, b, v, starts_of([L], gpu_device), scale=scale)
        s = torch.matmul(a[:, 0].double(), b[:, 0].double().t().contiguous()) * scale
        s = torch.where(torch.ones_like(s, dtype=torch.bool).tril_(), s, -math.inf)
        w = torch.softmax(s, 1)
        # rows whose weights do not hang on the rounding of a score: (d + 16) u of its size either way
        e = (d + 16) * U * torch.matmul(a[:, 0].double().abs(), b[:, 0].double().abs().t().contiguous()).amax(1) * scale
        top = torch.topk(s, 2, dim=1).values if L > 1 else s
        clear = (top[:, 0] - top[:, 1] > 2 * e + 40) | (e < 1e-3)
        clear[0] = True  # a key alone
        assert clear.sum() > 1 or size == 65504.0
        want_ = torch.matmul(w, v[:, 0].double())
        err = (out[:, 0].double() - want_).abs().amax(1)
        assert torch.all(torch.isfinite(out)) and torch.all(err[clear] <= 8 * H * float(v.abs().max()))


@pytest.mark.parametrize("count", [63, 64, 65, 130, 1000, 5000])
def test_many_sequences(K, gpu_device, count):
    r = np.random.default_rng(count)
    lengths = r.integers(0, 4, count).tolist()
    lengths[count // 3] = 150
    q, k, v = make(r, sum(lengths), 2, 1, 64, True, gpu_device)
    out = K.flash_attention_packed(q, k, v, starts_of(lengths, gpu_device))
    # each against the same rows on their own
    ends = np.cumsum(lengths)
    for s in {0, 1, 62, count // 3, count // 2, count - 2, count - 1}:
        rows = slice(int(ends[s]) - lengths[s], int(ends[s]))
        if lengths[s]:
            w, tol = want(q[rows], k[rows], v[rows], 0.125)
            assert torch.all((out[rows].double() - w).abs() <= tol), s
    ones = np.flatnonzero(np.array(lengths) == 1)
    rows = torch.from_numpy(ends[ones] - 1).to(gpu_device)
    assert torch.equal(out[rows], v[rows].expand(-1, 2, -1))  # a key alone has all the weight


def test_a_million_blocks(K, gpu_device):
    """More workgroups than a row of the grid has: every token a sequence, which gives its value."""
    count = 100000
    q, k, v = make(np.random.default_rng(25), count, 12, 12, 16, False, gpu_device)
    assert torch.equal(K.flash_attention_packed(q, k, v, torch.arange(count + 1, device=gpu_device)), v)


@pytest.mark.parametrize("heads", [3, 200])
@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
def test_hidden_keys_play_no_part(K, gpu_device, d, heads):
    """Infinities and NaN in later tokens, other sequences, and rows of none: the bits of finite ones there."""
    r = np.random.default_rng(10)
    lengths, first = [70, 33, 300, 1], 5
    total = first + sum(lengths) + 9
    q, k, v = (t.clone() for t in make(r, total, heads, heads, d, False, gpu_device))
    starts = starts_of(lengths, gpu_device, first)
    clean = K.flash_attention_packed(q, k, v, starts)
    end = first + sum(lengths)
    for bad in (math.nan, math.inf, -math.inf):
        a, b, c = q.clone(), k.clone(), v.clone()
        for t in (a, b, c):
            t[:first] = bad
            t[end:] = bad
        assert torch.equal(K.flash_attention_packed(a, b, c, starts)[first:end], clean[first:end])
        for spoilt in (first + 69, first + 70 + 20, first + 103 + 130, first + 103 + 255):
            for which in (1, 2):  # a key, a value
                x = [q, k.clone(), v.clone()]
                x[which][spoilt] = bad
                got = K.flash_attention_packed(*x, starts)
                s = int(torch.searchsorted(starts, spoilt, right=True)) - 1
                behind = torch.zeros(total, dtype=torch.bool, device=gpu_device)
                behind[spoilt:int(starts[s + 1])] = True
                there = torch.zeros_like(behind)
                there[first:end] = True
                fine = there & ~behind
                # the wavefronts that met it form their rows another way: roundings, not bits
                assert torch.all((got[fine].double() - clean[fine].double()).abs() <= 4 * H * clean[fine].double().abs() + 2e-3)
                far = fine.clone()
                far[spoilt - 63:spoilt] = False  # a tile of 64 keys may have both in it
                assert torch.equal(got[far], clean[far])
                if which == 2:
                    assert not torch.any(torch.isfinite(got[behind]))
                elif math.isnan(bad):
                    assert torch.all(torch.isnan(got[behind]))


@pytest.mark.parametrize("heads", [45, 100])
@pytest.mark.parametrize("d", [16, 32, 64])
def test_hidden_keys_in_every_deal(K, gpu_device, d, heads):
    test_hidden_keys_play_no_part(K, gpu_device, d, heads)


def test_many_numbers_that_are_none(K, gpu_device):
    """Long prompts in which every query meets one, or the last alone."""
    r = np.random.default_rng(22)
    L = 20000
    q, k, v = (t.clone() for t in make(r, L, 8, 2, 128, False, gpu_device))
    starts = starts_of([L], gpu_device)
    clean = K.flash_attention_packed(q, k, v, starts)
    for which in (0, 1, 2):
        x = [q.clone(), k.clone(), v.clone()]
        x[which][L - 1] = math.nan
        got = K.flash_attention_packed(*x, starts)
        assert torch.all(torch.isnan(got[L - 1])) and torch.equal(got[:L - 64], clean[:L - 64])
        x[which][:] = math.nan
        assert torch.all(torch.isnan(K.flash_attention_packed(*x, starts)))
    k[0] = math.nan
    assert torch.all(torch.isnan(K.flash_attention_packed(q, k, v, starts)))


def test_out_in_the_place_of_q(K, gpu_device):
    r = np.random.default_rng(23)
    for lengths in ([300, 1, 77], [2000, 3000]):
        q, k, v = make(r, sum(lengths), 12, 4, 64, False, gpu_device)
        starts = starts_of(lengths, gpu_device)
        apart = K.flash_attention_packed(q, k, v, starts)
        assert torch.equal(K.flash_attention_packed(q, k, v, starts, out=q), apart)


def test_rows_of_no_sequence_stay(K, gpu_device):
    r = np.random.default_rng(11)
    for d in (16, 64, 128, 256):
        q, k, v = make(r, 400, 4, 2, d, True, gpu_device)
        out = torch.full((400, 4, d), 7.0, dtype=torch.float16, device=gpu_device)
        got = K.flash_attention_packed(q, k, v, torch.tensor([100, 170, 170, 301], device=gpu_device), out=out)
        assert got is out and torch.all(out[:100] == 7) and torch.all(out[301:] == 7)
        w, tol = want(q[100:170], k[100:170], v[100:170], d ** -0.5)
        assert torch.all((out[100:170].double() - w).abs() <= tol)


def test_starts_that_are_wrong_reach_no_row_outside(K, gpu_device):
    r = np.random.default_rng(12)
    q, k, v = make(r, 300, 2, 2, 64, False, gpu_device)
    for starts in ([-50, 20, 300], [0, 200, 100, 300], [0, 100, 5000], [400, 500], [-10, -5], [10**12, 0, 300], [-10**12, 10**12]):
        buf = torch.full((302, 2, 64), 7.0, dtype=torch.float16, device=gpu_device)
        out = K.flash_attention_packed(q, k, v, torch.tensor(starts, device=gpu_device), out=buf[1:301])
        assert torch.all(buf[0] == 7) and torch.all(buf[301] == 7)
        assert torch.all(torch.isfinite(out))


def test_views_and_pitches(K, gpu_device):
    """Heads in front of rows, every other row, more than one token's room between rows."""
    r = np.random.default_rng(13)
    lengths = [77, 140]
    total = sum(lengths)
    q, k, v = make(r, total, 4, 2, 64, False, gpu_device)
    base = K.flash_attention_packed(q, k, v, starts_of(lengths, gpu_device))
    heads_first = tuple(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    assert torch.equal(K.flash_attention_packed(*heads_first, starts_of(lengths, gpu_device)), base)

    def spaced(t):
        big = torch.full((2 * total, t.shape[1], 64 + 8), math.nan, dtype=torch.float16, device=gpu_device)
        big[::2, :, 8:] = t
        return big[::2, :, 8:]

    assert torch.equal(K.flash_attention_packed(spaced(q), spaced(k), spaced(v), starts_of(lengths, gpu_device)), base)
    one_key_head = k[:, :1].expand(-1, 2, -1)  # a pitch of 0
    check(K, q, one_key_head, v, lengths)
    # one row, one head: no pitch at all
    odd = torch.randn(3, 1, 67, dtype=torch.float16, device=gpu_device)
    token = odd[:1, :, :64]
    check(K, token.expand(1, 4, 64), token, token, [1])


def test_rows_beyond_32_bits(K, gpu_device):
    r = np.random.default_rng(14)
    lengths = [200, 140, 60]
    total, pitch = sum(lengths), 12_000_000  # 400 rows: 4.8e9 elements
    buf = torch.empty((total - 1) * pitch + 3 * 64, dtype=torch.float16, device=gpu_device)
    y = buf.as_strided((total, 3, 64), (pitch, 64, 1))
    y.copy_(torch.from_numpy(r.standard_normal((total, 3, 64)).astype(np.float16)))
    check(K, y[:, :1], y[:, 1:2], y[:, 2:], lengths)


def test_equal_lengths_as_flash_attention_v1(K, gpu_device):
    r = np.random.default_rng(15)
    for B, n, L, d in ((3, 4, 200, 64), (2, 3, 77, 128)):
        q, k, v = make(r, B * L, n, n, d, True, gpu_device)
        got = check(K, q, k, v, [L] * B)
        batch = [t.reshape(B, L, n, d).transpose(1, 2).contiguous() for t in (q, k, v)]
        other = K.flash_attention_v1(*batch).transpose(1, 2).reshape(B * L, n, d)
        assert float((got.double() - other.double()).abs().max()) <= 4 * 2.0**-10 * float(other.abs().max())


def test_streams_and_graphs(K, gpu_device):
    """Captured once, replayed for other lengths: the starts are read on the GPU."""
    r = np.random.default_rng(16)
    q, k, v = make(r, 700, 12, 12, 64, True, gpu_device)
    starts = starts_of([300, 400, 0, 0], gpu_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = K.flash_attention_packed(q, k, v, starts)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, K.flash_attention_packed(q, k, v, starts))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K.flash_attention_packed(q, k, v, starts)
    for lengths in ([300, 400, 0, 0], [1, 1, 1, 697], [0, 0, 700, 0], [175] * 4):
        starts.copy_(starts_of(lengths, gpu_device))
        q.copy_(torch.randn_like(q))
        graph.replay()
        assert torch.equal(out, K.flash_attention_packed(q, k, v, starts))
        torch.cuda.synchronize()


def test_texts_scored_together(K, gpu_device):
    """A layer's operators on texts of different lengths: product, attention, projection, LM head, scores."""
    r = np.random.default_rng(17)
    lengths, width, heads, V = [40, 1, 100, 23], 256, 4, 1003
    total = sum(lengths)

    def weight(*shape):
        return torch.from_numpy((r.standard_normal(shape) / math.sqrt(shape[0])).astype(np.float16)).to(gpu_device)

    x = torch.from_numpy(r.standard_normal((total, width)).astype(np.float16)).to(gpu_device)
    w_qkv, w_proj, wte = weight(width, 3 * width), weight(width, width), weight(width, V).t().contiguous()
    starts = starts_of(lengths, gpu_device)
    y = K.fused_ffn(x, w_qkv)
    q, k, v = y.view(total, 3, heads, 64).unbind(1)
    z = K.flash_attention_packed(q, k, v, starts)
    hidden = K.fused_ffn(z.view(total, width), w_proj, residual=x)
    logits = K.lm_head(hidden, K.pack_lm_head(wte))
    tokens = torch.from_numpy(r.integers(0, V, total)).to(gpu_device)
    together = K.token_log_probs(logits, tokens, top=5)
    at = 0
    for L in lengths:  # each text on its own, by the operators for one length
        rows = slice(at, at + L)
        at += L
        a, b, c = K.matmul_and_split_qkv(x[rows].contiguous().view(1, L, width), w_qkv, None, heads)
        o = K.flash_attention_v1(a, b, c).transpose(1, 2).reshape(L, width).contiguous()
        h = K.fused_ffn(o, w_proj, residual=x[rows].contiguous())
        s = K.token_log_probs(K.lm_head(h, wte), tokens[rows], top=5)
        # both round attention, hidden state and logits to fp16 at the same places: a few steps of a logit (below 8)
        assert torch.all((s.log_probs - together.log_probs[rows]).abs() <= 8 * 8 * H)
