"""Refusals of flash_attention_packed: before any launch, so none of them needs a GPU."""
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


def call(lib, q=FAKE, k=FAKE, v=FAKE, out=FAKE, starts=FAKE, S=2, T=8, N=4, G=2, d=64, q_row=256, q_head=64, k_row=128,
         k_head=64, v_row=128, v_head=64, scale=0.125, dtype=1):
    return lib.gptmi_flash_attn_packed(q, k, v, out, starts, S, T, N, G, d, q_row, q_head, k_row, k_head, v_row, v_head,
                                       scale, dtype, None)


def test_refusals(lib):
    odd = ctypes.c_void_p(264)
    for args in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(starts=None), dict(S=0), dict(T=0),
                 dict(N=0), dict(G=0), dict(N=5), dict(d=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
                 dict(scale=math.inf), dict(scale=1e21), dict(scale=1e-21), dict(dtype=3), dict(q=odd), dict(k=odd), dict(v=odd), dict(out=odd),
                 dict(starts=ctypes.c_void_p(260)), dict(q_row=257), dict(k_head=4), dict(v_row=129)):
        assert call(lib, **args) == -1, args
        assert b"flash_attn_packed" in lib.gptmi_last_error()
    for args in (dict(dtype=0), dict(d=48), dict(q_row=(1 << 24) + 8), dict(k_row=-8), dict(v_head=(1 << 40) + 8),
                 dict(T=1 << 31), dict(S=1 << 31), dict(N=1 << 21, G=1), dict(S=1 << 30, N=1 << 10)):
        assert call(lib, **args) == -2, args


def test_operator_refuses():
    q, k = torch.zeros(8, 4, 64, dtype=torch.float16), torch.zeros(8, 2, 64, dtype=torch.float16)
    starts = torch.tensor([0, 3, 8])
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.flash_attention_packed(q, k, k, starts)
    for args, error in (((q, k, k[:7], starts), AssertionError), ((q[:, :3], k, k, starts), AssertionError),
                        ((q[:, :, :48], k[:, :, :48], k[:, :, :48], starts), AssertionError),
                        ((q, k, k, starts[:1]), AssertionError), ((q, k, k, starts.view(1, 3)), AssertionError),
                        ((q, k.float(), k, starts), TypeError), ((q, k, k, starts.int()), TypeError),
                        ((q.float(), k.float(), k.float(), starts), NotImplementedError),
                        ((q.bfloat16(), k.bfloat16(), k.bfloat16(), starts), TypeError),
                        ((q[:7], k, k, starts), AssertionError)):
        with pytest.raises(error):
            kernels.flash_attention_packed(*args)
