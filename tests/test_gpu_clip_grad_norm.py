"""clip_grad_norm_ against its formula in 64 bits: the norm, rounded once to fp32 (its sums' errors are some 2^-50), is off by
2^-24 of itself and as much again for a scale and a limit that are fp32 numbers, by 2^-150 at least (half a step of the
subnormal ones); a result by that of the factor (2^-24), of the
product (2^-24) and of its type (2^-11 in fp16, at least 2^-25)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16


@pytest.fixture(scope="module")
def K(gpu_device):
    from gpt_triton_amd import kernels

    return kernels


def want(grads, max_norm, scale):
    """(norm, results) in 64 bits of tensors."""
    total = sum(float(g.double().pow(2).sum()) for g in grads)
    norm = math.sqrt(total) * scale
    by = scale * (1.0 if norm <= max_norm else max_norm / norm)
    return norm, [g.double() * by for g in grads]


def check(K, grads, max_norm, scale=1.0, out=None):
    norm, results = want(grads, max_norm, scale)
    kept = [g.clone() for g in grads]
    got = K.clip_grad_norm_(grads, max_norm, scale=scale, out=out)
    assert got.shape == () and got.dtype == F32
    assert abs(float(got) - norm) <= 2.0**-23 * norm + 2.0**-150
    for o, w in zip(grads if out is None else out, results):
        half = o.dtype == F16
        assert torch.all((o.double() - w).abs() <= (2.0**-22 + (2.0**-11 if half else 0.0)) * w.abs() + (2.0**-25 if half else 2.0**-150))
    if out is not None:
        assert all(torch.equal(a, b) for a, b in zip(kept, grads) if not any(b.data_ptr() == o.data_ptr() for o in out))
    elif norm <= max_norm and scale == 1.0:
        assert all(torch.equal(a, b) for a, b in zip(kept, grads))
    return got


def make(shapes, dtype, device, spread=1.0, seed=0):
    r = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=r) * spread).to(device, dtype) for s in shapes]


SHAPES = [[(1,)], [(7,), (768,), (3, 5, 7)], [(300, 256), (256,), (0,), (1,), (64, 1000)], [(1025, 513)],
          [(4096,), (8192,), (8193,), (16384,)], [(n,) for n in range(1, 131)], [(5,)] * 300, [(1_500_007,), (3,), (2_000_000,)]]


@pytest.mark.parametrize("shapes", SHAPES, ids=range(len(SHAPES)))
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("max_norm", [0.5, 1e9, math.inf])
def test_in_place(K, gpu_device, shapes, dtype, max_norm):
    check(K, make(shapes, dtype, gpu_device), max_norm)


@pytest.mark.parametrize("shapes", SHAPES, ids=range(len(SHAPES)))
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("to", [F32, F16])
@pytest.mark.parametrize("max_norm,scale", [(0.5, 1.0), (1e9, 2.0**-10), (0.1, 1 / 3)])
def test_out(K, gpu_device, shapes, dtype, to, max_norm, scale):
    grads = make(shapes, dtype, gpu_device, 3.0)
    check(K, grads, max_norm, scale, [torch.full_like(g, math.nan, dtype=to) for g in grads])


def test_scale_in_place(K, gpu_device):
    check(K, make([(1000,), (33, 3)], F16, gpu_device, 100.0), 1e9, 1 / 64)


def test_mixed_types(K, gpu_device):
    grads = [g.to(F16 if n % 3 else F32) for n, g in enumerate(make([(100 + n,) for n in range(20)], F32, gpu_device))]
    check(K, [g.clone() for g in grads], 1.0)
    out = [torch.empty_like(g, dtype=F32 if n % 2 else F16) for n, g in enumerate(grads)]
    check(K, grads, 1.0, 0.5, out)
    some = [g if n % 2 else torch.empty_like(g) for n, g in enumerate(grads)]  # some in place
    check(K, grads, 1.0, 0.5, some)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("to", [F32, F16])
@pytest.mark.parametrize("at,to_at", [(1, 0), (0, 1), (1, 1), (3, 5), (7, 7), (2, 6)])
def test_addresses(K, gpu_device, dtype, to, at, to_at):
    """Views of a buffer at any element, with what lies around them left as it was."""
    for n in (1, 6, 50, 9000, 40_001):
        x, y = torch.randn(n + 16, device=gpu_device).to(dtype), torch.full((n + 16,), 7.0, device=gpu_device, dtype=to)
        check(K, [x[at:at + n]], 0.5, 1.0, [y[to_at:to_at + n]])
        assert torch.all(y[:to_at] == 7) and torch.all(y[to_at + n:] == 7)
        kept = x.clone()
        check(K, [x[at:at + n]], 0.5)
        assert torch.equal(x[:at], kept[:at]) and torch.equal(x[at + n:], kept[at + n:])


def test_orders_of_dimensions(K, gpu_device):
    a = torch.randn(40, 30, device=gpu_device).t()
    b = torch.randn(2, 5, 7, device=gpu_device).permute(2, 0, 1)
    check(K, [a, b], 0.5)
    check(K, [a, b], 0.1, 1.0, [torch.empty_like(a), torch.empty_like(b, dtype=F16)])


def test_sizes_of_numbers(K, gpu_device):
    """Squares beyond fp32's range on both sides."""
    for x in (2.0**100, 2.0**-100, 2.0**-147):
        check(K, [torch.full((5000,), x, device=gpu_device)], min(x, 1.0), 1.0, [torch.empty(5000, device=gpu_device)])
    g = torch.full((5000,), 3e38, device=gpu_device)
    norm = K.clip_grad_norm_([g], 1.0)
    assert float(norm) == math.inf  # beyond fp32, and the gradients are clipped all the same
    assert torch.all((g.double() - 1 / math.sqrt(5000)).abs() < 1e-8)
    zero = torch.zeros(100, device=gpu_device)
    assert float(K.clip_grad_norm_([zero], 1.0)) == 0.0 and not zero.any()
    tiny = torch.full((64,), 2.0**-24, device=gpu_device, dtype=F16)
    check(K, [tiny], 1.0, 1.0)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("at", [0, 4999, 77_777])
def test_infinities(K, gpu_device, dtype, bad, at):
    grads = make([(5000,), (72_778,)], dtype, gpu_device)
    flat = torch.cat(grads)
    flat[at] = bad
    grads = list(flat.split([5000, 72_778]))
    norm = K.clip_grad_norm_(grads, 1.0)
    if math.isnan(bad):
        assert math.isnan(float(norm)) and torch.isnan(flat).all()
    else:
        assert float(norm) == math.inf and math.isnan(float(flat[at]))
        flat[at] = 0.0
        assert not flat.any()


def test_same_bits_and_other_stream(K, gpu_device):
    grads = make([(100_000 + n,) for n in range(150)], F32, gpu_device)
    first = K.clip_grad_norm_(grads, math.inf)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = K.clip_grad_norm_(grads, math.inf)
    side.synchronize()
    assert torch.equal(first, again)


def test_largest(K, gpu_device):
    """More than 2^32 bytes in a tensor."""
    g = torch.ones(1_200_000_000, device=gpu_device, dtype=F32)
    g[-1] = 3.0
    norm = K.clip_grad_norm_([g], 2.0**10)
    w = math.sqrt(1_200_000_008.0)
    assert abs(float(norm) - w) <= 2.0**-23 * w
    by = 2.0**10 / w
    for part, x in ((g[:1000], 1.0), (g[-1001:-1], 1.0), (g[-1:], 3.0), (g[600_000_000:600_001_000], 1.0)):
        assert torch.all((part.double() - x * by).abs() <= 2.0**-22 * x * by)


def test_versions(K, gpu_device):
    g, o = torch.randn(10, device=gpu_device), torch.randn(10, device=gpu_device)
    before = g._version, o._version
    K.clip_grad_norm_([g], 1.0, out=[o])
    assert g._version == before[0] and o._version > before[1]
    K.clip_grad_norm_([g], 1.0)
    assert g._version > before[0]
    with torch.inference_mode():
        K.clip_grad_norm_([torch.randn(10, device=gpu_device)], 1.0)


def test_refusals(K, gpu_device):
    g, h = torch.randn(100, device=gpu_device), torch.randn(100, device=gpu_device)
    call = K.clip_grad_norm_
    for args, more, error in ((([],), {}, AssertionError), (([g.cpu()],), {}, RuntimeError), (([g, h.cpu()],), {}, RuntimeError),
                              (([g.double()],), {}, TypeError), (([g.bfloat16()],), {}, TypeError),
                              (([g[::2]],), {}, AssertionError), (([g[:1].expand(5)],), {}, AssertionError),
                              (([g, g],), {}, RuntimeError), (([g, g[50:]],), {}, RuntimeError),
                              (([g],), dict(out=[h, h]), AssertionError), (([g],), dict(out=[h[:50]]), AssertionError),
                              (([g[:50]],), dict(out=[g[25:75]]), RuntimeError), (([g, h],), dict(out=[h, g]), RuntimeError),
                              (([g[:50]],), dict(out=[g.view(torch.float16)[:50]]), RuntimeError),
                              (([g.view(10, 10).t()],), dict(out=[h.view(10, 10)]), AssertionError)):
        kept = g.clone(), h.clone()
        with pytest.raises(error):
            call(*args, 0.5, **more)
        assert torch.equal(g, kept[0]) and torch.equal(h, kept[1])
    for bad in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError):
            call([g], bad)
        with pytest.raises(ValueError):
            call([g], 1.0, scale=bad)
    with pytest.raises(ValueError):
        call([g], 1.0, scale=math.inf)
    with pytest.raises(RuntimeError, match="derivative"):
        call([g.clone().requires_grad_()], 1.0)
    with torch.no_grad():
        call([g.clone().requires_grad_()], 1.0)


def test_captured(K, gpu_device):
    grads = make([(1000 + 7 * n,) for n in range(130)], F16, gpu_device)
    out = [torch.empty_like(g, dtype=F32) for g in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.clip_grad_norm_(grads, 1.0, scale=0.5, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = K.clip_grad_norm_(grads, 1.0, scale=0.5, out=out)
    for n in range(3):
        for g, x in zip(grads, make([g.shape for g in grads], F16, gpu_device, 10.0**-n, 40 + n)):
            g.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        eager = [torch.empty_like(o) for o in out]
        assert torch.equal(norm, K.clip_grad_norm_(grads, 1.0, scale=0.5, out=eager))
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        check(K, grads, 1.0, 0.5, eager)


def test_nothing_to_clip(K, gpu_device):
    """Empty tensors alone, also more than a launch takes, and zeros."""
    empty = [torch.empty(0, 4, device=gpu_device, dtype=t) for t in (F32, F16) for _ in range(100)]
    assert float(K.clip_grad_norm_(empty, 1.0)) == 0.0
    zeros = [torch.zeros(5000, device=gpu_device)]
    assert float(K.clip_grad_norm_(empty + zeros, 1.0, scale=3.0)) == 0.0 and not zeros[0].any()


def test_out_in_place(K, gpu_device):
    """A gradient itself as its result, beside others that have one of their own."""
    grads = make([(300, 40), (7,), (20000,)], F32, gpu_device)
    wanted = want([g.clone() for g in grads], 0.5, 0.25)[1]
    kept = grads[1].clone()
    out = [grads[0], torch.empty(7, device=gpu_device, dtype=F16), grads[2]]
    K.clip_grad_norm_((g for g in grads), 0.5, scale=0.25, out=out)
    assert torch.equal(kept, grads[1])
    for o, w in zip(out, wanted):
        half = o.dtype == F16
        assert torch.all((o.double() - w).abs() <= (2.0**-22 + (2.0**-11 if half else 0.0)) * w.abs() + (2.0**-25 if half else 0.0))
