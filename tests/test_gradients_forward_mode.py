"""Embeddings, packed attention and clipping have no forward-mode derivative: a tensor with a tangent is refused, in front of
everything else, and no tangent is lost without a word."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from gpt_triton_amd import kernels as K


@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(requires_grad):
    ids, starts = torch.zeros(1, 4, dtype=torch.int64), torch.tensor([0, 4])
    q = torch.zeros(4, 2, 64, dtype=torch.float16, requires_grad=requires_grad)
    w = torch.zeros(8, 16, requires_grad=requires_grad)
    with forward_ad.dual_level():
        def dual(a):
            return forward_ad.make_dual(a, torch.ones_like(a))

        for call in (lambda: K.fused_embeddings(ids, dual(w), w), lambda: K.fused_embeddings(ids, w, dual(w)),
                     lambda: K.flash_attention_packed(dual(q), q, q, starts),
                     lambda: K.flash_attention_packed(q, q, dual(q), starts, out=torch.empty_like(q)),
                     lambda: K.clip_grad_norm_([w, dual(w)], 1.0), lambda: K.clip_grad_norm_([w], 1.0, out=[dual(w)])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        # without a tangent they go on, to the next refusal
        for call in (lambda: K.fused_embeddings(ids, w, w), lambda: K.flash_attention_packed(q, q, q, starts),
                     lambda: K.clip_grad_norm_([w], 1.0)):
            with pytest.raises(RuntimeError, match="GPU"):
                call()
