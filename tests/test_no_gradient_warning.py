"""Operators without a gradient say so where an activation requires one: gradients that reach it another way would lack their
part without a word.  The warning comes before anything else, so that these calls need no GPU."""
import warnings

import pytest
import torch

from gpt_triton_amd import kernels

W, B = torch.zeros(64, 64), torch.zeros(64)


def calls(x):
    heads = x.view(1, 1, 4, 64)
    flat = x.view(4, 1, 64).half()
    return {
        "fused_embeddings_layer_norm": lambda: kernels.fused_embeddings_layer_norm(torch.zeros(1, 4, dtype=torch.int64),
                                                                                   x.view(4, 64), W, B, B),
        "fused_layer_norm": lambda: kernels.fused_layer_norm(x, B, B),
        "fused_softmax": lambda: kernels.fused_softmax(x),
        "fused_ffn": lambda: kernels.fused_ffn(x, W),
        "fused_ffn, residual": lambda: kernels.fused_ffn(x.detach(), W, residual=x),
        "lm_head": lambda: kernels.lm_head(x, W),
        "matmul_and_split_qkv": lambda: kernels.matmul_and_split_qkv(x, torch.zeros(64, 192), None, 4),
        "flash_attention_v1": lambda: kernels.flash_attention_v1(heads, heads.detach(), heads.detach()),
        "attention_block": lambda: kernels.attention_block(x, B, B, torch.zeros(64, 192), torch.zeros(192), W, B, 1),
        "mlp_block": lambda: kernels.mlp_block(x, B, B, W, B, W, B),
        "block_layers": lambda: kernels.block_layers(x, [], 1, 64),
        "flash_attention_packed with out": lambda: kernels.flash_attention_packed(
            flat, flat, flat, torch.tensor([0, 4]), out=torch.zeros(4, 1, 64, dtype=torch.float16)),
    }


NAMES = list(calls(torch.zeros(1, 4, 64)))


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("leaf", [True, False])
def test_warns(name, leaf):
    x = torch.zeros(1, 4, 64, requires_grad=True)
    call = calls(x if leaf else x * 1.0)[name]
    with pytest.warns(UserWarning, match=f"{name.split(',')[0]} has no gradient") as met:
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    assert len(met) == 1 and met[0].filename == __file__


@pytest.mark.parametrize("name", NAMES)
def test_does_not_warn(name):
    x = torch.zeros(1, 4, 64, requires_grad=True)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with pytest.raises(RuntimeError, match="GPU only"):
            calls(x.detach())[name]()
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
            calls(x)[name]()


def test_weights_do_not_warn():
    x, w, b = torch.zeros(1, 4, 64), W.clone().requires_grad_(), B.clone().requires_grad_()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for call in (lambda: kernels.fused_ffn(x, w, b), lambda: kernels.fused_layer_norm(x, b, b),
                     lambda: kernels.lm_head(x, w)):
            with pytest.raises(RuntimeError, match="GPU only"):
                call()
