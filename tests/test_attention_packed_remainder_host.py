"""Refusals of the training forms of flash_attention_packed that keep a remainder: before any launch, so none of them needs a
GPU."""
import ctypes

import pytest

from test_attention_packed_grad_host import BEYOND, FAKE, SIZES, lib  # noqa: F401

ODD = ctypes.c_void_p(264)


def train(lib, q=FAKE, k=FAKE, v=FAKE, out=FAKE, stats=FAKE, remainder=FAKE, starts=FAKE, S=2, T=8, N=4, G=2, d=64, q_row=256,
          q_head=64, k_row=128, k_head=64, v_row=128, v_head=64, scale=0.125, dtype=1):
    return lib.gptmi_flash_attn_packed_train_remainder(q, k, v, out, stats, remainder, starts, S, T, N, G, d, q_row, q_head,
                                                       k_row, k_head, v_row, v_head, scale, dtype, None)


def backward(lib, q=FAKE, k=FAKE, v=FAKE, out=FAKE, stats=FAKE, remainder=FAKE, d_out=FAKE, starts=FAKE, dq=FAKE, dk=FAKE,
             dv=FAKE, S=2, T=8, N=4, G=2, d=64, q_row=256, q_head=64, k_row=128, k_head=64, v_row=128, v_head=64, scale=0.125,
             ws=FAKE, ws_bytes=1 << 20, dtype=1):
    return lib.gptmi_flash_attn_packed_backward_remainder(q, k, v, out, stats, remainder, d_out, starts, dq, dk, dv, S, T, N, G,
                                                          d, q_row, q_head, k_row, k_head, v_row, v_head, scale, ws, ws_bytes,
                                                          dtype, None)


@pytest.mark.parametrize("call,more", [(train, ()), (backward, ("d_out",))])
def test_refusals(lib, call, more):  # noqa: F811
    for args in (*SIZES, *(dict([(n, x)]) for n in ("q", "k", "v", "out", "remainder", *more) for x in (None, ODD)),
                 dict(stats=None), dict(stats=ctypes.c_void_p(260)), dict(starts=None), dict(starts=ctypes.c_void_p(260))):
        assert call(lib, **args) == -1, args
        assert f"flash_attn_packed_{call.__name__}_remainder" in lib.gptmi_last_error().decode()
    for args in (*BEYOND[:4], dict(N=1 << 21, G=1), dict(S=1, T=40, N=1 << 20, d=32)):
        assert call(lib, **args) == -2, args
    if call is backward:
        needed = lib.gptmi_flash_attn_packed_backward_workspace_bytes(2, 8, 4, 2, 64)
        for args in (dict(ws=None), dict(ws_bytes=needed - 1), dict(ws=ODD)):
            assert call(lib, **args) == -3, args
