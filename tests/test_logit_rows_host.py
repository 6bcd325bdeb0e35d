"""Refusals of token_log_probs and distillation_loss: before any launch, so none of them needs a GPU."""
import ctypes
import math
import os

import pytest
import torch

from gpt_triton_amd import _lib, kernels


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from gpt_triton_amd import build

        build.build()
    return _lib.load()


FAKE = ctypes.c_void_p(256)  # never dereferenced: the refusal comes first


def scores(lib, x=FAKE, ld=64, tokens=FAKE, tau=1.0, lp=FAKE, ent=FAKE, top=0, top_lp=None, top_t=None, M=4, V=64,
           dtype=1):
    return lib.gptmi_token_log_probs(x, ld, tokens, tau, lp, ent, top, top_lp, top_t, M, V, dtype, None)


def test_scores_refusals(lib):
    bad = [dict(x=None), dict(ld=-1), dict(tau=0.0), dict(tau=-1.0), dict(tau=math.nan), dict(tau=math.inf),
           dict(M=0), dict(V=0), dict(dtype=2), dict(tokens=None), dict(top=-1), dict(top=65, top_lp=FAKE, top_t=FAKE),
           dict(top=5), dict(top=5, top_lp=FAKE), dict(lp=None, ent=None), dict(x=ctypes.c_void_p(257)),
           dict(x=ctypes.c_void_p(258), dtype=0)]
    for args in bad:
        assert scores(lib, **args) == -1, args
        assert b"token_log_probs" in lib.gptmi_last_error()
    beyond = [dict(top=129, top_lp=FAKE, top_t=FAKE, V=1000, ld=1000), dict(M=1 << 31), dict(V=(1 << 30) + 1),
              dict(ld=(1 << 40) + 1)]
    for args in beyond:
        assert scores(lib, **args) == -2, args


def test_gradient_refusals(lib):
    def call(x=FAKE, ld=64, tokens=FAKE, tau=1.0, g=FAKE, g_pitch=1, h=None, h_pitch=1, top=0, ids=None, u=None, grad=FAKE, ld_grad=64, M=4,
             V=64, dtype=1):
        return lib.gptmi_token_log_probs_backward(x, ld, tokens, tau, g, g_pitch, h, h_pitch, top, ids, u, grad, ld_grad, M, V, dtype,
                                                  None)

    for args in (dict(x=None), dict(grad=None), dict(ld_grad=63), dict(tokens=None), dict(top=3), dict(top=3, ids=FAKE),
                 dict(grad=ctypes.c_void_p(257)), dict(tau=0.0), dict(top=-1), dict(g_pitch=2), dict(h_pitch=-1)):
        assert call(**args) == -1, args
    assert call(top=129, ids=FAKE, u=FAKE) == -2
    assert call(ld_grad=(1 << 40) + 1) == -2


def test_distillation_refusals(lib):
    def call(x=FAKE, ld=64, ids=FAKE, t=FAKE, k=4, tau=1.0, d=None, d_pitch=1, losses=FAKE, grad=None, ld_grad=64, M=4, V=64, dtype=1,
             t_dtype=0):
        return lib.gptmi_distillation_loss(x, ld, ids, t, k, tau, None, d, d_pitch, losses, grad, ld_grad, M, V, dtype, t_dtype,
                                           None)

    for args in (dict(x=None), dict(ids=None), dict(t=None), dict(k=0), dict(losses=None), dict(t_dtype=2),
                 dict(t=ctypes.c_void_p(258)), dict(grad=FAKE, ld_grad=63), dict(tau=-1.0), dict(dtype=-1), dict(d_pitch=4)):
        assert call(**args) == -1, args
    assert call(k=129) == -2


def test_operators_refuse_the_cpu():
    x, t = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64)
    ids, teacher = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    for call in (lambda: kernels.token_log_probs(x, t), lambda: kernels.token_log_probs(x.requires_grad_(), t),
                 lambda: kernels.distillation_loss(x, ids, teacher),
                 lambda: kernels.distillation_loss_and_grad(x, ids, teacher)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_only_the_logits_have_a_gradient():
    x, ids = torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(AssertionError):
        kernels.distillation_loss(x, ids, torch.zeros(2, 3, requires_grad=True))
    with pytest.raises(AssertionError):
        kernels.distillation_loss_and_grad(x, ids, torch.zeros(2, 3), 1.0, torch.ones(2, requires_grad=True))
