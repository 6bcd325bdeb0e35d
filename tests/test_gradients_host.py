"""Refusals of gptmi_embed_backward and gptmi_clip_grad_norm: before any launch, so none of them needs a GPU."""
import array
import ctypes
import math
import os

import pytest
import torch

from gpt_triton_amd import _lib, kernels

FAKE = ctypes.c_void_p(256)  # never dereferenced: the refusal comes first


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from gpt_triton_amd import build

        build.build()
    return _lib.load()


def embed(lib, ids=FAKE, dz=FAKE, d_wte=FAKE, d_wpe=FAKE, B=2, L=300, V=100, P=300, H=64, p=0.0, ws=FAKE, ws_bytes=1 << 30,
          dtype=1):
    return lib.gptmi_embed_backward(ids, dz, d_wte, d_wpe, B, L, V, P, H, p, 1337, ws, ws_bytes, dtype, None)


def test_embed_backward(lib):
    for args in (dict(ids=None), dict(dz=None), dict(d_wte=None, d_wpe=None), dict(B=0), dict(L=0), dict(V=0), dict(P=0),
                 dict(H=0), dict(P=299), dict(dtype=2), dict(p=1.0), dict(p=-0.1), dict(p=math.nan),
                 dict(dz=ctypes.c_void_p(257)), dict(d_wte=ctypes.c_void_p(258), dtype=0), dict(ids=ctypes.c_void_p(260))):
        assert embed(lib, **args) == -1, args
        assert b"embed_backward" in lib.gptmi_last_error()
    for args in (dict(B=1 << 30), dict(V=(1 << 26) + 1), dict(P=(1 << 24) + 1), dict(H=(1 << 20) + 1), dict(B=1 << 62)):
        assert embed(lib, **args) == -2, args
    needed = lib.gptmi_embed_backward_workspace_bytes(2, 300, 64)
    assert needed > 0 and lib.gptmi_embed_backward_workspace_bytes(1, 256, 64) == 0
    for args in (dict(ws=None), dict(ws_bytes=needed - 1), dict(ws=ctypes.c_void_p(264))):
        assert embed(lib, **args) == -3, args
    for args in ((0, 3, 4), (3, 0, 4), (3, 3, 0), (1 << 30, 3, 4), (1 << 62, 3, 4), (2, 2, 1 << 21)):
        assert lib.gptmi_embed_backward_workspace_bytes(*args) == 0


def test_tables_beyond_the_grid(lib):
    """The token table's zero rows are a workgroup of 1024 threads for each 64 KB: below 2^32 threads."""
    for args in (dict(V=1 << 26, H=1 << 10), dict(V=(1 << 24) + 1, H=1 << 10), dict(V=1 << 20, H=1 << 20, P=300)):
        assert embed(lib, **args, ws=None) == -2, args
    assert embed(lib, V=1 << 24, H=1 << 10, ws=None) == -3


def clip(lib, grads=(4096,), out=None, sizes=(100,), f16=(0,), out_f16=None, n=None, scale=1.0, max_norm=1.0, norm=FAKE, ws=FAKE,
         ws_bytes=1 << 20):
    at = array.array("Q", grads)
    to = array.array("Q", grads if out is None else out)
    count = array.array("q", sizes)
    return lib.gptmi_clip_grad_norm(at.buffer_info()[0], to.buffer_info()[0], count.buffer_info()[0], bytes(f16),
                                    bytes(f16 if out_f16 is None else out_f16), len(grads) if n is None else n, scale, max_norm,
                                    norm, ws, ws_bytes, None)


def test_clip_grad_norm(lib):
    two = dict(sizes=(100, 100), f16=(0, 0))
    for args in (dict(n=0), dict(n=-1), dict(norm=None), dict(norm=ctypes.c_void_p(258)), dict(scale=0.0), dict(scale=-1.0),
                 dict(scale=math.inf), dict(scale=math.nan), dict(max_norm=0.0), dict(max_norm=math.nan), dict(max_norm=-1.0),
                 dict(grads=(0,)), dict(grads=(4098,)), dict(grads=(4097,), f16=(1,)), dict(sizes=(-1,)), dict(sizes=(1 << 43,)),
                 dict(out=(0,)), dict(out=(8194,)),
                 # the same twice, one inside another, results over gradients and each other
                 dict(grads=(4096, 4096), **two), dict(grads=(4096, 4492), **two), dict(grads=(4492, 4096), **two),
                 dict(grads=(4096, 4100), sizes=(100, 1), f16=(0, 0)), dict(out=(4100,)), dict(out=(4096,), out_f16=(1,)),
                 dict(grads=(4096, 8192), out=(8192, 4096), **two), dict(grads=(4096, 8192), out=(16384, 16780), **two),
                 dict(grads=(4096, 8192), out=(4096, 4492), **two)):
        assert clip(lib, **args) == -1, args
        assert b"clip_grad_norm" in lib.gptmi_last_error()
    assert clip(lib, n=(1 << 20) + 1) == -2
    needed = lib.gptmi_clip_grad_norm_workspace_bytes(1)
    for args in (dict(ws=None), dict(ws_bytes=needed - 1), dict(ws=ctypes.c_void_p(260))):
        assert clip(lib, **args) == -3, args
    for n in (0, -1, (1 << 20) + 1):
        assert lib.gptmi_clip_grad_norm_workspace_bytes(n) == 0


def test_operators_refuse():
    x, w = torch.zeros(1, 4, dtype=torch.int64), torch.zeros(8, 16, requires_grad=True)
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.fused_embeddings(x, w, w)
    with pytest.raises(TypeError):
        kernels.fused_embeddings(x.int(), w, w)
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.clip_grad_norm_([torch.zeros(4)], 1.0)
    with pytest.raises(AssertionError):
        kernels.clip_grad_norm_([], 1.0)


def test_orders_without_gaps():
    t = torch.zeros(4, 6, 5)
    for x, fine in ((t, True), (t.permute(2, 0, 1), True), (t.transpose(0, 1), True), (t[:, :3], False), (t[:, :, ::2], False),
                    (t[:1].expand(4, 6, 5), False), (t[:1].transpose(0, 2), True), (torch.zeros(()), True), (torch.zeros(0, 3), True),
                    (t[0].t(), True), (t[:, 0], False), (t.as_strided((3, 3), (1, 2)), False)):
        assert kernels._side_by_side(x) == fine
