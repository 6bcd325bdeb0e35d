"""Gradients of fused_embeddings against their formula.

Whole numbers are summed without rounding, so those are compared bit by bit (fp16: rounded once at the end).  For others a
sum of n numbers in fp32 is off by at most n 2^-24 times the sum of their sizes, and the result by half a step of its type
(2^-24 or 2^-11 of itself, at least 2^-25 in fp16)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16]


@pytest.fixture(scope="module")
def K(gpu_device):
    from gpt_triton_amd import kernels

    return kernels


def want(ids, dz, V, P, dtype=np.float64):
    """(d_wte, d_wpe) in 64 bits; ids outside [0, V) have a place alone."""
    B, L, H = dz.shape
    d_wte, d_wpe = np.zeros((V, H), dtype), np.zeros((P, H), dtype)
    rows = dz.reshape(-1, H).astype(dtype)
    flat = ids.reshape(-1)
    known = (flat >= 0) & (flat < V)
    np.add.at(d_wte, flat[known], rows[known])
    d_wpe[:L] = dz.astype(dtype).sum(0)
    return d_wte, d_wpe


def grads(K, ids, dz, V, P, device, dropout_prob=0.0):
    dz = dz if torch.is_tensor(dz) else torch.from_numpy(dz).to(device)
    ids = ids if torch.is_tensor(ids) else torch.from_numpy(ids).to(device)
    H = dz.shape[2]
    r = torch.Generator().manual_seed(1)
    wte = torch.randn(V, H, generator=r).to(device, dz.dtype).requires_grad_()
    wpe = torch.randn(P, H, generator=r).to(device, dz.dtype).requires_grad_()
    z = K.fused_embeddings(ids, wte, wpe, dropout_prob)
    assert torch.equal(z, K.fused_embeddings(ids, wte.detach(), wpe.detach(), dropout_prob))
    got = torch.autograd.grad(z, (wte, wpe), dz)
    for g, like in zip(got, (wte, wpe)):
        assert g.shape == like.shape and g.dtype == like.dtype and g.is_contiguous()
    return got


def texts(r, B, L, V):
    """Tokens some of which are far more frequent than others, the first and the last among them."""
    ids = np.minimum((np.exp(r.random((B, L)) * np.log(V + 1)) - 1).astype(np.int64), V - 1)
    ids = (ids * 7919) % V
    ids[0, 0], ids[-1, -1] = 0, V - 1
    return ids


def exact(K, device, B, L, V, P, H, dtype, seed=0, ids=None):
    r = np.random.default_rng(seed)
    ids = texts(r, B, L, V) if ids is None else ids
    dz = r.integers(-4, 5, (B, L, H)).astype(np.float32)
    got = grads(K, ids, torch.from_numpy(dz).to(device, dtype), V, P, device)
    for g, w in zip(got, want(ids, dz, V, P, np.float32)):
        assert torch.equal(g, torch.from_numpy(w).to(device, dtype)), (B, L, V, H)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,L", [(1, 1), (1, 24), (2, 64), (1, 255), (4, 64), (257, 1), (1, 300), (3, 1000), (4, 1024),
                                 (1, 4097), (64, 130)])
@pytest.mark.parametrize("V,H", [(1, 8), (2, 64), (300, 256), (511, 100), (512, 33), (50257, 48)])
def test_whole_numbers(K, gpu_device, B, L, V, H, dtype):
    exact(K, gpu_device, B, L, V, L + 3, H, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H", [1, 2, 7, 16, 255, 256, 260, 768, 1000, 1024, 1032, 1600, 2048, 2056, 4100, 8200])
@pytest.mark.parametrize("B,L", [(2, 70), (3, 120)])
def test_widths(K, gpu_device, H, B, L, dtype):
    exact(K, gpu_device, B, L, 1000, 128, H, dtype)


@pytest.mark.parametrize("V", [65535, 65536, 128256, 262143, 262144, 1 << 22])
@pytest.mark.parametrize("B,L", [(2, 100), (5, 999)])
def test_vocabularies(K, gpu_device, V, B, L):
    exact(K, gpu_device, B, L, V, 1024, 8, torch.float16)


@pytest.mark.parametrize("B,L", [(32, 1024), (127, 300), (512, 300), (300, 1023)])
def test_many_tokens(K, gpu_device, B, L):
    exact(K, gpu_device, B, L, 50257, 1024, 16, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,L", [(1, 200), (7, 500), (150, 900)])
def test_one_token(K, gpu_device, B, L, dtype):
    """All positions, and all but a few, have the same one."""
    r = np.random.default_rng(4)
    ids = np.full((B, L), 17, np.int64)
    sign = np.where(np.arange(B * L) % 2, 1, -1).reshape(B, L, 1).astype(np.float32)
    for n in (0, 3):
        ids.reshape(-1)[r.integers(0, B * L, n)] = 5
        dz = np.broadcast_to(sign, (B, L, 24)).copy()
        got = grads(K, ids, torch.from_numpy(dz).to(gpu_device, dtype), 40, L, gpu_device)
        for g, w in zip(got, want(ids, dz, 40, L)):
            assert torch.equal(g, torch.from_numpy(w).to(gpu_device, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,L", [(2, 60), (9, 300)])
def test_unknown_tokens(K, gpu_device, B, L, dtype):
    r = np.random.default_rng(5)
    ids = texts(r, B, L, 200)
    ids[r.random((B, L)) < 0.3] = -100
    ids[r.random((B, L)) < 0.1] = 200
    ids[0, 1], ids[0, 2] = 2**40 + 3, -(2**62)
    exact(K, gpu_device, B, L, 200, L, 64, dtype, ids=ids)
    exact(K, gpu_device, B, L, 200, L, 64, dtype, ids=np.full((B, L), -1, np.int64))


@pytest.mark.parametrize("dtype,half_step", [(torch.float32, 2.0**-24), (torch.float16, 2.0**-11)])
@pytest.mark.parametrize("B,L,V,H", [(2, 64, 50257, 768), (8, 512, 3000, 320), (64, 300, 50257, 96)])
def test_numbers(K, gpu_device, B, L, V, H, dtype, half_step):
    r = np.random.default_rng(6)
    ids = texts(r, B, L, V)
    dz = torch.from_numpy(r.standard_normal((B, L, H)).astype(np.float32)).to(dtype)
    got = grads(K, ids, dz.to(gpu_device), V, L, gpu_device)
    x = dz.double().numpy()
    count = np.bincount(ids.reshape(-1), minlength=V)[:, None]
    for g, w, size, n in zip(got, want(ids, x, V, L), want(ids, abs(x), V, L), (count, B)):
        tol = n * 2.0**-24 * size + half_step * abs(w) + (2.0**-25 if dtype == torch.float16 else 0.0)
        assert np.all(abs(g.double().cpu().numpy() - w) <= tol)


@pytest.mark.parametrize("dtype,half_step", [(torch.float32, 2.0**-24), (torch.float16, 2.0**-11)])
@pytest.mark.parametrize("B,L,H", [(2, 64, 768), (5, 200, 100), (3, 200, 33)])
def test_dropout(K, gpu_device, B, L, H, dtype, half_step):
    """The forward pass's mask, one for all rows, over 1 - p."""
    r = np.random.default_rng(7)
    ids, p = texts(r, B, L, 500), 0.25
    dz = r.integers(-4, 5, (B, L, H)).astype(np.float32)
    one = K.fused_embeddings(torch.zeros(1, 1, dtype=torch.int64, device=gpu_device),
                             torch.ones(1, H, device=gpu_device), torch.zeros(1, H, device=gpu_device), p)
    kept = (one != 0).view(-1).cpu().numpy()
    assert 0 < kept.sum() < H
    got = grads(K, ids, torch.from_numpy(dz).to(gpu_device, dtype), 500, L, gpu_device, p)
    for g, w in zip(got, want(ids, dz, 500, L)):
        w = np.where(kept, w / 0.75, 0.0)
        assert np.all(abs(g.double().cpu().numpy() - w) <= (half_step + 2.0**-23) * abs(w))


def test_some_of_the_gradients(K, gpu_device):
    r = np.random.default_rng(8)
    for B, L in ((2, 50), (6, 200)):
        ids = torch.from_numpy(texts(r, B, L, 100)).to(gpu_device)
        dz = torch.from_numpy(r.integers(-4, 5, (B, L, 32)).astype(np.float32)).to(gpu_device)
        both = grads(K, ids, dz, 100, L + 1, gpu_device)
        wte, wpe = torch.randn(100, 32, device=gpu_device), torch.randn(L + 1, 32, device=gpu_device)
        for a, b in ((True, False), (False, True)):
            tables = wte.clone().requires_grad_(a), wpe.clone().requires_grad_(b)
            got, = torch.autograd.grad(K.fused_embeddings(ids, *tables), [t for t in tables if t.requires_grad], dz)
            assert torch.equal(got, both[0] if a else both[1])
        assert not K.fused_embeddings(ids, wte, wpe).requires_grad
        with torch.no_grad():
            assert not K.fused_embeddings(ids, wte.requires_grad_(), wpe).requires_grad


def test_forms_of_the_gradient(K, gpu_device):
    """One number for all of it, columns of something wider, an odd address."""
    r = np.random.default_rng(9)
    for B, L in ((2, 50), (6, 200)):
        ids = texts(r, B, L, 100)
        dz = torch.from_numpy(r.integers(-4, 5, (B, L, 32)).astype(np.float32)).to(gpu_device)
        both = grads(K, ids, dz, 100, L, gpu_device)
        wide = torch.zeros(B, L, 40, device=gpu_device)
        wide[..., 3:35] = dz
        odd = torch.zeros(dz.numel() + 1, device=gpu_device)[1:].view(dz.shape)
        odd.copy_(dz)
        for x in (wide[..., 3:35], odd):
            assert all(torch.equal(a, b) for a, b in zip(both, grads(K, ids, x, 100, L, gpu_device)))
        ones = grads(K, ids, torch.ones_like(dz), 100, L, gpu_device)
        one = grads(K, ids, torch.ones((), device=gpu_device).expand(dz.shape), 100, L, gpu_device)
        assert all(torch.equal(a, b) for a, b in zip(ones, one))


def test_same_bits_and_other_stream(K, gpu_device):
    r = np.random.default_rng(10)
    ids = torch.from_numpy(texts(r, 16, 500, 1000)).to(gpu_device)
    dz = torch.from_numpy(r.standard_normal((16, 500, 128)).astype(np.float32)).to(gpu_device)
    first = grads(K, ids, dz, 1000, 512, gpu_device)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = grads(K, ids, dz, 1000, 512, gpu_device)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_infinities_stay_with_their_tokens(K, gpu_device):
    for B, L in ((1, 8), (3, 200)):
        ids = np.arange(B * L).reshape(B, L)
        dz = np.ones((B, L, 16), np.float32)
        dz[0, 5, 3] = np.inf
        dz[0, 6, 2] = np.nan
        d_wte, d_wpe = grads(K, ids, dz, B * L, L, gpu_device)
        for g in (d_wte, d_wpe):
            bad = torch.nonzero(~torch.isfinite(g)).tolist()
            assert bad == [[5, 3], [6, 2]]


def test_derivatives_that_there_are_not(K, gpu_device):
    ids = torch.zeros(1, 4, dtype=torch.int64, device=gpu_device)
    w = torch.randn(4, 8, device=gpu_device).requires_grad_()
    z = K.fused_embeddings(ids, w, w)
    with pytest.raises(RuntimeError, match="first derivative"):
        torch.autograd.grad(z.sum(), w, create_graph=True)


@pytest.mark.parametrize("B,L", [(2, 100), (4, 300)])
def test_captured_step(K, gpu_device, B, L):
    r = np.random.default_rng(11)
    ids = torch.from_numpy(texts(r, B, L, 700)).to(gpu_device)
    dz = torch.randn(B, L, 64, device=gpu_device)
    tables = torch.randn(700, 64, device=gpu_device).requires_grad_(), torch.randn(L, 64, device=gpu_device).requires_grad_()

    def step():
        z = K.fused_embeddings(ids, *tables)
        return (z, *torch.autograd.grad(z, tables, dz))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in range(3):
        ids.copy_(torch.from_numpy(texts(np.random.default_rng(30 + n), B, L, 700)))
        dz.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got[1:], grads(K, ids.clone(), dz.clone(), 700, L, gpu_device)):
            assert torch.equal(a, b)


def test_largest(K, gpu_device):
    """More than 2^32 bytes and 2^31 elements of the output's gradient: whole numbers, summed without rounding."""
    B, L, V, H = 2100, 1024, 50257, 1032
    r = torch.Generator(device=gpu_device).manual_seed(3)
    ids = torch.randint(0, V, (B, L), device=gpu_device, generator=r)
    dz = torch.randint(-4, 5, (B, L, H), device=gpu_device, generator=r, dtype=torch.int8).half()
    got = grads(K, ids, dz, V, L, gpu_device)
    d_wte, d_wpe = (torch.zeros(n, H, device=gpu_device) for n in (V, L))
    for i in range(0, B, 100):
        rows = dz[i:i + 100].float()
        d_wte.index_add_(0, ids[i:i + 100].reshape(-1), rows.view(-1, H))
        d_wpe += rows.sum(0)
    for g, w in zip(got, (d_wte, d_wpe)):
        assert torch.equal(g, w.half())


def test_two_streams_at_once(K, gpu_device):
    r = np.random.default_rng(22)
    ids = [torch.from_numpy(texts(r, 40, 300, 1000)).to(gpu_device) for _ in range(2)]
    dz = [torch.randn(40, 300, 256, device=gpu_device).half() for _ in range(2)]
    alone = [grads(K, i, x, 1000, 300, gpu_device) for i, x in zip(ids, dz)]
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(3):
        for n, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[n].append(grads(K, ids[n], dz[n], 1000, 300, gpu_device))
    torch.cuda.synchronize()
    for n in range(2):
        for one in got[n]:
            assert all(torch.equal(a, b) for a, b in zip(one, alone[n]))


@pytest.mark.parametrize("B,L,more", [(4097, 1, 0), (1, 4097, 1), (5461, 3, 1000), (8, 2048, 0), (16385, 1, 70), (2, 150, 3000)])
@pytest.mark.parametrize("V,H", [(50257, 40), (600, 33), (1 << 18, 8)])
def test_where_the_sort_changes(K, gpu_device, B, L, more, V, H):
    """A workgroup that sorts all tokens, of 4 or of 16 a thread, and tiles of them; rows of the position table that no token
    has are zeros, whole blocks of them and parts."""
    for dtype in DTYPES:
        exact(K, gpu_device, B, L, V, L + more, H, dtype)


def test_one_token_in_a_large_tile(K, gpu_device):
    for n in (4098, 16384):
        exact(K, gpu_device, n // 2, 2, 1000, 2, 24, torch.float32, ids=np.full((n // 2, 2), 999))
