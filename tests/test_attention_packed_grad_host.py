"""Refusals of the training forms of flash_attention_packed: before any launch, so none of them needs a GPU."""
import ctypes
import math
import os

import numpy as np
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


def train(lib, q=FAKE, k=FAKE, v=FAKE, out=FAKE, stats=FAKE, starts=FAKE, S=2, T=8, N=4, G=2, d=64, q_row=256, q_head=64,
          k_row=128, k_head=64, v_row=128, v_head=64, scale=0.125, dtype=1):
    return lib.gptmi_flash_attn_packed_train(q, k, v, out, stats, starts, S, T, N, G, d, q_row, q_head, k_row, k_head, v_row,
                                             v_head, scale, dtype, None)


def backward(lib, q=FAKE, k=FAKE, v=FAKE, out=FAKE, stats=FAKE, d_out=FAKE, starts=FAKE, dq=FAKE, dk=FAKE, dv=FAKE, S=2, T=8,
             N=4, G=2, d=64, q_row=256, q_head=64, k_row=128, k_head=64, v_row=128, v_head=64, scale=0.125, ws=FAKE,
             ws_bytes=1 << 20, dtype=1):
    return lib.gptmi_flash_attn_packed_backward(q, k, v, out, stats, d_out, starts, dq, dk, dv, S, T, N, G, d, q_row, q_head,
                                                k_row, k_head, v_row, v_head, scale, ws, ws_bytes, dtype, None)


SIZES = (dict(S=0), dict(T=0), dict(N=0), dict(G=0), dict(N=5), dict(d=0), dict(scale=0.0), dict(scale=math.nan),
         dict(scale=1e21), dict(dtype=3), dict(q_row=257), dict(k_head=4), dict(v_row=129))
BEYOND = (dict(dtype=0), dict(q_row=(1 << 24) + 8), dict(k_row=-8), dict(v_head=(1 << 40) + 8), dict(T=1 << 31),
          dict(S=1 << 31), dict(N=1 << 21, G=1))


def test_refusals(lib):
    odd = ctypes.c_void_p(264)
    for args in (*SIZES, *(dict([(n, x)]) for n in ("q", "k", "v", "out") for x in (None, odd)), dict(stats=None),
                 dict(stats=ctypes.c_void_p(260)), dict(starts=None), dict(starts=ctypes.c_void_p(260))):
        assert train(lib, **args) == -1, args
        assert b"flash_attn_packed_train" in lib.gptmi_last_error()
    for args in (*SIZES, *(dict([(n, x)]) for n in ("q", "k", "v", "out", "d_out") for x in (None, odd)), dict(dq=odd),
                 dict(dk=odd), dict(dv=odd), dict(dk=None), dict(dv=None), dict(dq=None, dk=None, dv=None), dict(stats=None),
                 dict(stats=ctypes.c_void_p(260)), dict(starts=None), dict(starts=ctypes.c_void_p(260))):
        assert backward(lib, **args) == -1, args
        assert b"flash_attn_packed_backward" in lib.gptmi_last_error()
    for args in (*BEYOND, dict(d=48)):
        assert train(lib, **args) == -2, args
    for args in (*BEYOND[:4], dict(N=1 << 21, G=1)):
        assert backward(lib, **args) == -2, args
    needed = lib.gptmi_flash_attn_packed_backward_workspace_bytes(2, 8, 4, 2, 64)
    for args in (dict(ws=None), dict(ws_bytes=needed - 1), dict(ws=ctypes.c_void_p(264))):
        assert backward(lib, **args) == -3, args
    for args in ((0, 8, 4, 2, 64), (2, 0, 4, 2, 64), (2, 8, 0, 2, 64), (2, 8, 4, 0, 64), (2, 8, 5, 2, 64), (2, 8, 4, 2, 0),
                 (2, 1 << 31, 4, 2, 64), (2, 8, 1 << 21, 1, 64), (1 << 31, 8, 4, 2, 64)):
        assert lib.gptmi_flash_attn_packed_backward_workspace_bytes(*args) == 0


def test_rows_of_the_output(lib):
    """Offsets inside a tile of rows of the output and its gradient are 32-bit numbers."""
    for n, d in ((1 << 20, 256), (1 << 20, 32), ((1 << 18) + 2, 64), ((1 << 16) + 2, 256)):
        sizes = dict(S=1, T=40, N=n, d=d)
        assert train(lib, **sizes) == -2, sizes
        assert backward(lib, **sizes, ws=None) == -2, sizes
    for n, d in ((1 << 20, 16), (1 << 18, 64), (1 << 16, 256)):
        assert backward(lib, S=1, T=40, N=n, d=d, ws=None) == -3


def test_operator_refuses():
    q, k = (torch.zeros(8, n, 64, dtype=torch.float16, requires_grad=True) for n in (4, 2))
    starts = torch.tensor([0, 3, 8])
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.flash_attention_packed(q, k, k, starts)
    for args, error in (((q, k, k[:7], starts), AssertionError), ((q, k.float(), k, starts), TypeError),
                        ((q.float(), k.float(), k.float(), starts), NotImplementedError)):
        with pytest.raises(error):
            kernels.flash_attention_packed(*args)


def test_formula_against_differences():
    """The formula that the gradients are held to, in 64 bits: each gradient against differences of the output."""
    r = np.random.default_rng(0)
    L, d, scale = 6, 4, 0.7
    q, k, v, e = (torch.from_numpy(r.standard_normal((L, d))) for _ in range(4))
    past = torch.ones(L, L, dtype=torch.bool).tril_()

    def loss(q, k, v):
        return (torch.softmax(torch.where(past, q @ k.T * scale, -math.inf), 1) @ v * e).sum()

    w = torch.softmax(torch.where(past, q @ k.T * scale, -math.inf), 1)
    p = e @ v.T
    x = w * (p - (w @ v * e).sum(1, keepdim=True)) * scale
    for n, got in enumerate((x @ k, x.T @ q, w.T @ e)):
        for i in range(L):
            for j in range(d):
                step = torch.zeros(L, d, dtype=torch.float64)
                step[i, j] = 1e-5
                ends = [loss(*[t + s * step if m == n else t for m, t in enumerate((q, k, v))]) for s in (1, -1)]
                # the third derivative's part, some 1e-10, and the rounding of a difference over 2e-5
                assert abs(float(got[i, j]) - float(ends[0] - ends[1]) / 2e-5) < 1e-8
