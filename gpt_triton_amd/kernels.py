"""Operator layer: the five public functions of the reference's kernels.py, with the same
names, argument order, defaults, assertions and return shapes, each handing raw device
pointers to one entry point of libgptmi.so (include/gptmi.h).

    fused_embeddings(x, wte, wpe, dropout_prob=0.0)              kernels.py:75-101
    fused_layer_norm(x, weight, bias)                            kernels.py:148-164
    fused_ffn(x, weight, bias=None, residual=None,
              add_gelu=False, dropout_prob=0.0)                  kernels.py:260-315
    matmul_and_split_qkv(x, weight, bias, num_heads)             kernels.py:347-367
    flash_attention_v1(q, k, v, dropout_prob=0.0)                kernels.py:477-525

plus `fused_embeddings_layer_norm` (the embedding gather and the first block's LayerNorm in one
kernel, the fusion the reference's author notes as a TODO, kernels.py:132-133), `fused_softmax(x)` (the reference only sketches a row softmax, kernels.py:318-342),
`lm_head(x, wte)` (the transposed-weight product the reference leaves as a TODO,
gpt.py:159-161) and `pack_weight(weight)`: the GEMM reads its weight as an fp16,
K-contiguous image, which `fused_ffn` / `matmul_and_split_qkv` otherwise rebuild on every call
where the kernels cannot read the weight in place (fp16, K a multiple of 64); a `PackedWeight` may be passed wherever they take `weight`.
For scoring texts and learning from the scores, which the reference has nothing for: `flash_attention_packed` (prompts of different
lengths without padding, grouped heads), `token_log_probs` (of rows of logits, with entropy, alternatives and gradient) and
`distillation_loss` / `distillation_loss_and_grad` (against a teacher's top logits).  `flash_attention_packed` and
`fused_embeddings` have gradients, and `clip_grad_norm_` clips all gradients together; the other operators have none, and warn
where an activation that they are given requires one (what their weights require is left alone).  Tensors must live on the
GPU: there is no CPU path.  dropout_prob > 0 reproduces the reference's masks: Philox-4x32-10
(Triton's tl.rand) with the kernels' default seed 1337 and the reference's offsets -- the column
for the embedding, the flat index m*N + n for fused_ffn, query*Lk + key for the attention
weights (kernels.py:31-34, 65-70, 245-251, 457-460).
"""
import array
import collections
import math
import os
import warnings

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.GPTMI_F32, torch.float16: _lib.GPTMI_F16}


def _dtype_code(t, what):
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"{what}: dtype {t.dtype} is not supported (float32 and float16 are)")


def _on_gpu(first, *rest):
    """Index of the GPU that all the tensors (None allowed behind the first) are on."""
    index = first.get_device()  # -1 on the CPU
    if index < 0:
        raise RuntimeError("gpt_triton_amd operators run on the GPU only; got a tensor on "
                           f"{first.device} (there is no CPU fallback)")
    for t in rest:
        if t is not None and t.get_device() != index:
            raise RuntimeError(f"tensors on different devices: {first.device} and {t.device}")
    return index


def _call(index, what, fn, *args):
    """One entry point of the library on torch's current stream of GPU `index`.  A forward of a few
    tokens is bound by the host: no device guard where the GPU is the current one already, the raw
    stream from torch's own binding instead of a torch.cuda.Stream object."""
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        _lib.check(rc, what)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(nbytes, like):
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def _no_gradient(what, stacklevel=3):
    """Of an operator without a gradient, called with an activation that requires one.  Its result is in no graph, so a backward
    pass by the activation's other uses, a residual's for one, ends without an error and without this operator's part."""
    if torch.is_grad_enabled():
        warnings.warn(f"{what} has no gradient: its result is cut off from its input, and gradients that reach the input another "
                      "way lack what would flow through here.  detach() the input, or use torch's operators, to say which is "
                      "meant", stacklevel=stacklevel)


class PackedWeight:
    """The fp16 [N][round_up(K, 64)] image of a [K, N] weight (see gptmi_pack_weight).  `shape`
    and `dtype` are those of the weight it was made from, so it can stand in for it."""

    __slots__ = ("data", "shape", "dtype", "device", "vocab")

    def __init__(self, data, shape, dtype, vocab=None):
        self.data, self.shape, self.dtype, self.device = data, tuple(shape), dtype, data.device
        self.vocab = vocab  # pack_lm_head: rows of wte before the zero padding

    def is_contiguous(self):
        return True

    def get_device(self):
        return self.data.get_device()

    def data_ptr(self):
        return self.data.data_ptr()


@torch.no_grad()
def pack_weight(weight):
    """Packs a contiguous [K, N] weight once; the result replaces `weight` in `fused_ffn` and
    `matmul_and_split_qkv` and must be rebuilt when the weight changes."""
    assert weight.dim() == 2 and weight.is_contiguous()
    dev = _on_gpu(weight)
    K_, N = weight.shape
    lib = _lib.load()
    buf = weight.new_empty(lib.gptmi_packed_weight_bytes(N, K_), dtype=torch.uint8)
    _call(dev, "pack_weight", lib.gptmi_pack_weight, weight.data_ptr(), buf.data_ptr(), N, K_,
          _lib.GPTMI_W_KN, _dtype_code(weight, "pack_weight"))
    return PackedWeight(buf, weight.shape, weight.dtype)


@torch.no_grad()
def pack_lm_head(wte):
    """Packs wte [V, H] once for `lm_head`, with the vocabulary padded to a multiple of 64 by zero
    rows.  GPT-2's V = 50257 is odd: rows of a dense [T, V] fp16 matrix then start on 2-byte
    boundaries and every logit is stored on its own.  With the padded image the GEMM writes
    [T, Vp] rows of whole 128-byte lines -- the shape the persistent GEMM kernel takes -- and
    `lm_head` returns the [.., :V] view of it."""
    assert wte.dim() == 2 and wte.is_contiguous()
    dev = _on_gpu(wte)
    V, H = wte.shape
    Vp = -(-V // 64) * 64
    lib = _lib.load()
    buf = wte.new_zeros(lib.gptmi_packed_weight_bytes(Vp, H), dtype=torch.uint8)
    _call(dev, "pack_lm_head", lib.gptmi_pack_weight, wte.data_ptr(), buf.data_ptr(), V, H,
          _lib.GPTMI_W_NK, _dtype_code(wte, "pack_lm_head"))
    return PackedWeight(buf, (H, Vp), wte.dtype, vocab=V)


def check_token_ids(x, vocab_size):
    """Raises IndexError if a token id lies outside [0, vocab_size).  The embedding kernels
    themselves read no memory for such an id and use a zero wte row (the reference reads out of
    bounds); this check costs a device synchronisation, so the operators run it only when the
    environment variable GPTMI_CHECK_IDS is set to 1."""
    lo, hi = int(x.min()), int(x.max())
    if lo < 0 or hi >= vocab_size:
        raise IndexError(f"token ids span [{lo}, {hi}] but the vocabulary has {vocab_size} rows")


def _maybe_check_ids(x, vocab_size):
    if os.environ.get("GPTMI_CHECK_IDS") == "1" and x.numel() > 0:
        check_token_ids(x, vocab_size)


def _wlayout(weight, default):
    return _lib.GPTMI_W_PACKED if isinstance(weight, PackedWeight) else default


def _embeddings(x, wte, wpe, dropout_prob):
    assert wte.shape[1] == wpe.shape[1]
    assert x.is_contiguous()
    assert wte.is_contiguous()
    assert wpe.is_contiguous()
    B, L = x.shape
    V, H = wte.shape
    P = wpe.shape[0]
    if x.dtype != torch.int64:
        raise TypeError(f"fused_embeddings: token ids must be int64, got {x.dtype}")
    if wte.dtype != wpe.dtype:
        raise TypeError("fused_embeddings: wte and wpe must share a dtype")
    dev = _on_gpu(x, wte, wpe)
    _maybe_check_ids(x, V)
    z = wte.new_empty((B, L, H))
    _call(dev, "fused_embeddings", _lib.load().gptmi_embed, x.data_ptr(), wte.data_ptr(),
          wpe.data_ptr(), z.data_ptr(), B, L, V, P, H, float(dropout_prob), 1337,
          _dtype_code(wte, "fused_embeddings"))
    return z


class _EmbeddingsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wte, wpe, dropout_prob):
        ctx.save_for_backward(x)
        ctx.tables, ctx.dropout_prob = (wte.shape[0], wpe.shape[0], wte.shape[1]), float(dropout_prob)
        return _embeddings(x, wte, wpe, dropout_prob)

    @staticmethod
    def backward(ctx, dz):
        _first_derivative("fused_embeddings")
        x, = ctx.saved_tensors
        (B, L), (V, P, H) = x.shape, ctx.tables
        dz = dz.contiguous()
        d_wte = dz.new_empty((V, H)) if ctx.needs_input_grad[1] else None
        d_wpe = dz.new_empty((P, H)) if ctx.needs_input_grad[2] else None
        lib = _lib.load()
        nbytes = 0 if d_wte is None else lib.gptmi_embed_backward_workspace_bytes(B, L, H)
        ws = _workspace(nbytes, dz)
        _call(dz.get_device(), "fused_embeddings", lib.gptmi_embed_backward, x.data_ptr(), dz.data_ptr(), _ptr(d_wte),
              _ptr(d_wpe), B, L, V, P, H, ctx.dropout_prob, 1337, _ptr(ws), nbytes, _dtype_code(dz, "fused_embeddings"))
        return None, d_wte, d_wpe, None


def fused_embeddings(x, wte, wpe, dropout_prob=0.0):
    """dropout(wte[x] + wpe[position]) for token ids x [B, L] -> [B, L, H] in wte's dtype.

    Gradients flow to wte and wpe, dense, backward and once: sums over a token's positions and over the batch, in fp32, each
    in one order, so that the same step gives the same bits."""
    _no_tangents("fused_embeddings", wte, wpe)
    if (wte.requires_grad or wpe.requires_grad) and torch.is_grad_enabled():
        return _EmbeddingsFunction.apply(x, wte, wpe, dropout_prob)
    return _embeddings(x, wte, wpe, dropout_prob)


def _side_by_side(t):
    """Whether a tensor's elements fill its memory without gaps, in whatever order of the dimensions."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((stride, size) for stride, size in zip(t.stride(), t.shape) if size != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def clip_grad_norm_(grads, max_norm, scale=1.0, out=None):
    """norm = scale * sqrt(sum of the squares of all elements of all of `grads`), and min(1, max_norm / norm) * scale times each
    gradient in its place, or in `out`'s tensor of the same shape (which leaves `grads` as they are).  Returns the norm, a
    float32 number on the GPU; nothing waits for it.

    grads: tensors, float32 or float16, on one GPU, dense in any order of dimensions, none twice; out: as many, each of
    either type and of the order of its gradient, none of which overlaps anything else; a gradient itself may be in its place.
    scale: the inverse of a loss scale; max_norm infinity: the norm, and the gradients times scale.  Squares are summed in 64
    bits.  Gradients in place are written only where the factor is not 1.  An infinity among them makes the norm infinite and
    the results 0 or NaN, a NaN makes all of them NaN: a step to skip.  With max_norm infinity, scale 1 and all in place the
    call is for the norm alone, which then is all that says so: no gradient is written, whatever it holds."""
    what = "clip_grad_norm_"
    grads = list(grads)
    outs = grads if out is None else list(out)
    assert grads, "no gradients"
    assert len(outs) == len(grads), (len(outs), len(grads))
    _no_tangents(what, *grads, *outs)
    dev = _on_gpu(*grads) if out is None else _on_gpu(*grads, *outs)
    scale, max_norm = float(scale), float(max_norm)
    if not 0.0 < scale < math.inf or not max_norm > 0.0:
        raise ValueError(f"{what}: scale {scale} or max_norm {max_norm} is not positive")
    every = grads if out is None else grads + outs
    types = [t.dtype for t in every]
    if not _DTYPES.keys() >= set(types):
        for t in every:
            _dtype_code(t, what)
    for t in every:
        assert t.is_contiguous() or _side_by_side(t), "the elements of a gradient must fill its memory"
    if torch.is_grad_enabled() and any([t.requires_grad for t in every]):
        raise RuntimeError(f"{what} has no derivative")
    if out is not None:
        for g, o in zip(grads, outs):
            assert o.shape == g.shape and (o.stride() == g.stride() or o.is_contiguous() and g.is_contiguous()), (
                "out must have the gradients' shapes and orders")
    n = len(grads)
    addresses = array.array("Q", [t.data_ptr() for t in every])
    sizes = array.array("q", [t.numel() for t in grads])
    halves = bytes([t is torch.float16 for t in types])
    at = addresses.buffer_info()[0]
    norm = grads[0].new_empty((), dtype=torch.float32)
    lib = _lib.load()
    nbytes = lib.gptmi_clip_grad_norm_workspace_bytes(n)
    ws = _workspace(nbytes, norm)
    _call(dev, what, lib.gptmi_clip_grad_norm, at, at if out is None else at + 8 * n, sizes.buffer_info()[0], halves,
          halves if out is None else halves[n:], n, scale, max_norm, norm.data_ptr(), _ptr(ws), nbytes)
    torch.autograd.graph.increment_version(outs)
    return norm


def fused_embeddings_layer_norm(x, wte, wpe, weight, bias):
    """(fused_embeddings(x, wte, wpe), fused_layer_norm(of that, weight, bias)) from one kernel:
    the embedding row is normalised while it is still in registers.  Both results are
    bit-identical to the two separate calls.  No dropout (eval-mode forward), and no gradients."""
    if wte.requires_grad or wpe.requires_grad:
        _no_gradient("fused_embeddings_layer_norm")
    assert wte.shape[1] == wpe.shape[1]
    assert x.is_contiguous()
    assert wte.is_contiguous()
    assert wpe.is_contiguous()
    assert weight.is_contiguous()
    assert bias.is_contiguous()
    assert weight.shape == bias.shape
    assert wte.shape[1] == weight.shape[0]
    B, L = x.shape
    V, H = wte.shape
    P = wpe.shape[0]
    if x.dtype != torch.int64:
        raise TypeError(f"fused_embeddings_layer_norm: token ids must be int64, got {x.dtype}")
    if not (wte.dtype == wpe.dtype == weight.dtype == bias.dtype):
        raise TypeError("fused_embeddings_layer_norm: wte, wpe, weight and bias must share a dtype")
    dev = _on_gpu(x, wte, wpe, weight, bias)
    _maybe_check_ids(x, V)
    emb = wte.new_empty((B, L, H))
    out = wte.new_empty((B, L, H))
    _call(dev, "fused_embeddings_layer_norm", _lib.load().gptmi_embed_layernorm, x.data_ptr(),
          wte.data_ptr(), wpe.data_ptr(), weight.data_ptr(), bias.data_ptr(), emb.data_ptr(),
          out.data_ptr(), B, L, V, P, H, 1e-5, _dtype_code(wte, "fused_embeddings_layer_norm"))
    return emb, out


def fused_layer_norm(x, weight, bias):
    """LayerNorm over the last dim (eps = 1e-5, biased variance), same shape and dtype as x."""
    if x.requires_grad:
        _no_gradient("fused_layer_norm")
    assert x.is_contiguous()
    assert weight.is_contiguous()
    assert bias.is_contiguous()
    assert weight.shape == bias.shape
    assert x.shape[-1] == weight.shape[0]
    if not (x.dtype == weight.dtype == bias.dtype):
        raise TypeError("fused_layer_norm: x, weight and bias must share a dtype")
    dev = _on_gpu(x, weight, bias)
    H = x.shape[-1]
    M = x.numel() // H
    z = torch.empty_like(x)
    _call(dev, "fused_layer_norm", _lib.load().gptmi_layernorm, x.data_ptr(), weight.data_ptr(),
          bias.data_ptr(), z.data_ptr(), M, H, 1e-5, _dtype_code(x, "fused_layer_norm"))
    return z


def fused_softmax(x):
    """softmax over the last dim with fp32 statistics, same shape and dtype as x."""
    if x.requires_grad:
        _no_gradient("fused_softmax")
    assert x.is_contiguous()
    dev = _on_gpu(x)
    H = x.shape[-1]
    M = x.numel() // H
    z = torch.empty_like(x)
    _call(dev, "fused_softmax", _lib.load().gptmi_softmax, x.data_ptr(), z.data_ptr(), M, H,
          _dtype_code(x, "fused_softmax"))
    return z


def _linear_workspace(lib, M, N, K, code, wlayout, like):
    """(workspace or None, its bytes).  A packed image under fp16 rows that are whole 128-byte lines
    needs none; that is every product of an eval-mode forward, and not worth a call to be told."""
    if wlayout == _lib.GPTMI_W_PACKED and code == _lib.GPTMI_F16 and K % 64 == 0:
        return None, 0
    nbytes = lib.gptmi_linear_workspace_bytes(M, N, K, code, wlayout)
    return _workspace(nbytes, like), nbytes


def _linear(x, weight, bias, residual, z, gelu, dropout_prob, wlayout, what):
    K, N = x.shape[-1], z.shape[-1]
    M = x.numel() // K
    dtype = x.dtype
    code = _dtype_code(x, what)
    if weight.dtype != dtype:
        raise TypeError(f"{what}: weight is {weight.dtype} but x is {dtype}")
    if bias is not None and bias.dtype != dtype:
        raise TypeError(f"{what}: bias is {bias.dtype} but x is {dtype}")
    if residual is not None and residual.dtype != dtype:
        raise TypeError(f"{what}: residual is {residual.dtype} but x is {dtype}")
    lib = _lib.load()
    ws, ws_bytes = _linear_workspace(lib, M, N, K, code, wlayout, x)
    _call(x.get_device(), what, lib.gptmi_linear, x.data_ptr(), weight.data_ptr(), _ptr(bias),
          _ptr(residual), z.data_ptr(), M, N, K, 1 if gelu else 0, float(dropout_prob), 1337, wlayout,
          _ptr(ws), ws_bytes, code)
    return z


def fused_ffn(x, weight, bias=None, residual=None, add_gelu=False, dropout_prob=0.0):
    """dropout(gelu?(x @ weight + bias)) + residual; weight is [K, N] (in x out)."""
    if x.requires_grad or residual is not None and residual.requires_grad:
        _no_gradient("fused_ffn")
    shape = x.shape
    K = shape[-1]
    N = weight.shape[1]
    _on_gpu(x, weight, bias, residual)
    z = x.new_empty((*shape[:-1], N))

    assert x.is_contiguous()
    assert weight.is_contiguous()
    assert K == weight.shape[0]
    if bias is not None:
        assert bias.is_contiguous()
        assert N == bias.shape[0]
    if residual is not None:
        assert residual.numel() == z.numel()
        assert residual.is_contiguous()

    return _linear(x, weight, bias, residual, z, add_gelu, dropout_prob,
                   _wlayout(weight, _lib.GPTMI_W_KN), "fused_ffn")


def lm_head(x, wte):
    """x @ wte^T: logits [*, V].  `wte` is the [V, H] embedding matrix itself (read in place, no
    transposed copy; the result is contiguous) or its `pack_lm_head` image (the result is then
    the [*, :V] view of a buffer whose rows are padded to a multiple of 64 logits)."""
    if x.requires_grad:
        _no_gradient("lm_head")
    shape = x.shape
    H = shape[-1]
    assert x.is_contiguous()
    assert wte.is_contiguous()
    _on_gpu(x, wte)
    if isinstance(wte, PackedWeight):
        assert wte.vocab is not None and H == wte.shape[0]
        z = x.new_empty((*shape[:-1], wte.shape[1]))
        _linear(x, wte, None, None, z, False, 0.0, _lib.GPTMI_W_PACKED, "lm_head")
        return z[..., :wte.vocab]
    assert H == wte.shape[1]
    z = x.new_empty((*shape[:-1], wte.shape[0]))
    return _linear(x, wte, None, None, z, False, 0.0, _lib.GPTMI_W_NK, "lm_head")


# Top tokens a row of `token_log_probs`, and a teacher's logits a row of `distillation_loss`.
MAX_TOP = 128

TokenLogProbs = collections.namedtuple("TokenLogProbs", "log_probs entropy top_log_probs top_tokens")


def _logit_rows(logits, what):
    """(GPU, type code, rows, vocabulary, pitch) of logits [.., V] whose rows lie at one pitch, as `lm_head` returns
    them: dense, or the front of padded rows."""
    dev = _on_gpu(logits)
    code = _dtype_code(logits, what)
    V = logits.shape[-1]
    assert V > 0 and (V == 1 or logits.stride(-1) == 1), "the logits of a row must lie side by side"
    rows = logits.numel() // V
    if rows <= 1:  # whatever its pitch is
        return dev, code, rows, V, V
    if logits.dim() == 2:
        return dev, code, rows, V, logits.stride(0)
    try:
        return dev, code, rows, V, logits.view(-1, V).stride(0)
    except RuntimeError:
        raise AssertionError(f"{what}: the rows of the logits must lie at one pitch") from None


def _logit_gradient(logits, rows, V, ld):
    """(a buffer for the gradient of rows of logits in their shape, its pitch).  Pitch and address equal the logits'
    modulo 64 elements and 16 bytes, so that the kernels read and write in the same chunks."""
    pitch = V + (ld - V) % 64
    offset = logits.data_ptr() % 16 // logits.element_size()
    if offset == 0 and (pitch == V or rows <= 1):
        return torch.empty_like(logits) if ld == V else logits.new_empty(logits.shape), pitch
    buf = logits.new_empty(offset + max(rows - 1, 0) * pitch + V)
    return buf.as_strided((rows, V), (pitch, 1), offset).view(logits.shape), pitch


def _check_row_tokens(t, shape, what):
    if t.dtype != torch.int64:
        raise TypeError(f"{what}: token ids must be int64, got {t.dtype}")
    assert t.shape == shape, (t.shape, shape)
    assert t.is_contiguous()


def _maybe_check_row_tokens(t, V, what):
    if os.environ.get("GPTMI_CHECK_IDS") == "1" and t.numel() > 0 and int(t.max()) >= V:
        raise IndexError(f"{what}: token id {int(t.max())}, but a row has {V} logits")


def _check_temperature(temperature, code, what):
    # the kernels' fp16 exponents are off by what fp32 rounds off the largest logit over the temperature
    least = 1e-4 if code == _lib.GPTMI_F16 else 1e-30
    if not least <= temperature <= 1e30:
        raise ValueError(f"{what}: temperature {temperature} is not between {least} and 1e30")


def _token_log_probs(logits, tokens, top, temperature):
    dev, code, rows, V, ld = _logit_rows(logits, "token_log_probs")
    lead = logits.shape[:-1]
    _on_gpu(logits, tokens)
    if tokens is not None:
        _check_row_tokens(tokens, lead, "token_log_probs")
        _maybe_check_row_tokens(tokens, V, "token_log_probs")
    assert 0 <= top <= V, (top, V)
    if top > MAX_TOP:
        raise NotImplementedError(f"token_log_probs: at most {MAX_TOP} top tokens, got {top}")
    _check_temperature(temperature, code, "token_log_probs")
    entropy = logits.new_empty(lead, dtype=torch.float32)
    log_probs = None if tokens is None else torch.empty_like(entropy)
    top_log_probs = top_tokens = None
    if top > 0:
        top_log_probs = entropy.new_empty((*lead, top))
        top_tokens = torch.empty_like(top_log_probs, dtype=torch.int64)
    if rows > 0:
        _call(dev, "token_log_probs", _lib.load().gptmi_token_log_probs, logits.data_ptr(), ld, _ptr(tokens),
              temperature, _ptr(log_probs), entropy.data_ptr(), top, _ptr(top_log_probs), _ptr(top_tokens), rows, V,
              code)
    return log_probs, entropy, top_log_probs, top_tokens


def _first_derivative(what):
    # in a backward pass autograd is on where the pass is itself to be differentiated
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} has a first derivative only")


def _no_tangents(what, *tensors):
    # the calls that leave torch's graph alone would drop them; a level of dual tensors is rarely open
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} has no forward-mode derivative")


def _row_gradient(g):
    """(address, pitch in rows, what to keep until the call) of a gradient with an element a row; autograd hands one
    number for all rows on as a view of pitch 0."""
    if g is None:
        return None, 0, None
    if not any(g.stride()):
        return g.data_ptr(), 0, g
    g = g.contiguous()
    return g.data_ptr(), 1, g


class _TokenLogProbsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, temperature):
        log_probs, entropy, top_log_probs, top_tokens = _token_log_probs(logits, tokens, top, temperature)
        ctx.set_materialize_grads(False)
        if top_tokens is not None:
            ctx.mark_non_differentiable(top_tokens)
        ctx.save_for_backward(logits, tokens, top_tokens)
        ctx.temperature = temperature
        return log_probs, entropy, top_log_probs, top_tokens

    @staticmethod
    def backward(ctx, d_log_probs, d_entropy, d_top, _):
        _first_derivative("token_log_probs")
        logits, tokens, top_tokens = ctx.saved_tensors
        if d_log_probs is None and d_entropy is None and d_top is None:
            return None, None, None, None
        dev, code, rows, V, ld = _logit_rows(logits, "token_log_probs")
        token_at, token_pitch, d_log_probs = _row_gradient(d_log_probs)
        entropy_at, entropy_pitch, d_entropy = _row_gradient(d_entropy)
        top = 0
        if d_top is not None:
            top, d_top = top_tokens.shape[-1], d_top.contiguous()
        grad, pitch = _logit_gradient(logits, rows, V, ld)
        if rows > 0:
            _call(dev, "token_log_probs_backward", _lib.load().gptmi_token_log_probs_backward, logits.data_ptr(), ld,
                  _ptr(tokens), ctx.temperature, token_at, token_pitch, entropy_at, entropy_pitch, top, _ptr(top_tokens),
                  _ptr(d_top), grad.data_ptr(), pitch, rows, V, code)
        return grad, None, None, None


def token_log_probs(logits, tokens=None, top=0, temperature=1.0):
    """Scores of rows of logits [.., V], as `lm_head` returns them, under softmax(logits / temperature):

        log_probs      [..]       the log probability of tokens [..]; a token outside [0, V), such as the -100 of
                                  padding, scores 0; None without tokens
        entropy        [..]       of the row's distribution
        top_log_probs  [.., top]  the `top` most likely tokens, the likeliest first, equal ones in the order of their
        top_tokens     [.., top]  ids, at most MAX_TOP; None for top = 0

    fp32 (the tokens int64, contiguous) whatever the logits' type.  Logits of -infinity mark tokens that cannot occur, and a
    row with a NaN, which is -infinity among the top tokens, or +infinity scores NaN.  Gradients flow to the logits from
    all but top_tokens, backward and once.  temperature from 1e-4 on (fp32 logits: 1e-30) to 1e30."""
    _no_tangents("token_log_probs", logits)
    temperature = float(temperature)
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogProbs(*_TokenLogProbsFunction.apply(logits, tokens, top, temperature))
    return TokenLogProbs(*_token_log_probs(logits, tokens, top, temperature))


def _distillation(logits, teacher_tokens, teacher_logits, temperature, weights, losses, gradient, d_losses=None):
    """(losses or None, gradient or None)."""
    what = "distillation_loss"
    dev, code, rows, V, ld = _logit_rows(logits, what)
    k = teacher_tokens.shape[-1]
    teacher_code = _dtype_code(teacher_logits, what)
    if d_losses is None:  # the forward pass of a gradient has checked these
        lead = logits.shape[:-1]
        _on_gpu(logits, teacher_tokens, teacher_logits, weights)
        _check_row_tokens(teacher_tokens, (*lead, k), what)
        _maybe_check_row_tokens(teacher_tokens, V, what)
        assert teacher_logits.shape == teacher_tokens.shape, (teacher_logits.shape, teacher_tokens.shape)
        assert teacher_logits.is_contiguous()
        assert k > 0
        if k > MAX_TOP:
            raise NotImplementedError(f"{what}: at most {MAX_TOP} of the teacher's logits a row, got {k}")
        if weights is not None:
            if weights.dtype != torch.float32:
                raise TypeError(f"{what}: weights must be float32, got {weights.dtype}")
            assert weights.shape == lead, (weights.shape, lead)
            assert weights.is_contiguous()
        _check_temperature(temperature, code, what)
    out = None
    if losses:
        out = logits.new_empty(lead, dtype=torch.float32) if weights is None else torch.empty_like(weights)
    grad, pitch = _logit_gradient(logits, rows, V, ld) if gradient else (None, V)
    d_at, d_pitch, d_losses = _row_gradient(d_losses)
    if rows > 0:
        _call(dev, what, _lib.load().gptmi_distillation_loss, logits.data_ptr(), ld, teacher_tokens.data_ptr(),
              teacher_logits.data_ptr(), k, temperature, _ptr(weights), d_at, d_pitch, _ptr(out), _ptr(grad), pitch, rows,
              V, code, teacher_code)
    return out, grad


class _DistillationFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_tokens, teacher_logits, temperature, weights):
        ctx.save_for_backward(logits, teacher_tokens, teacher_logits, weights)
        ctx.temperature = temperature
        return _distillation(logits, teacher_tokens, teacher_logits, temperature, weights, True, False)[0]

    @staticmethod
    def backward(ctx, d_losses):
        _first_derivative("distillation_loss")
        logits, teacher_tokens, teacher_logits, weights = ctx.saved_tensors
        grad = _distillation(logits, teacher_tokens, teacher_logits, ctx.temperature, weights, False, True, d_losses)[1]
        return grad, None, None, None, None


def _check_derivatives(logits, *constants):
    assert not any(t is not None and t.requires_grad for t in constants), "only the logits have a gradient"
    _no_tangents("distillation_loss", logits, *constants)


def distillation_loss(logits, teacher_tokens, teacher_logits, temperature=1.0, weights=None):
    """Losses [..] (fp32) of a student's logits [.., V] against a teacher's top logits: with q the softmax of
    teacher_logits [.., k] / temperature (float32 or float16; log probabilities serve as well) and p that of logits /
    temperature,

        weights * sum_i q_i (log q_i - log p[teacher_tokens_i])

    k up to MAX_TOP; all but the logits contiguous.  An entry whose token is outside [0, V) or whose logit is -infinity
    counts for nothing; a row without entries has loss and gradient 0, whatever its logits are.  weights [..] (float32, all
    1 if None): 0 marks padding, whose logits may be anything.  Gradients flow to the logits alone, which are read again
    for them, backward and once; `distillation_loss_and_grad` has both in one pass.  temperature as in
    `token_log_probs`."""
    _check_derivatives(logits, teacher_logits, weights)
    temperature = float(temperature)
    if logits.requires_grad and torch.is_grad_enabled():
        return _DistillationFunction.apply(logits, teacher_tokens, teacher_logits, temperature, weights)
    return _distillation(logits, teacher_tokens, teacher_logits, temperature, weights, True, False)[0]


def distillation_loss_and_grad(logits, teacher_tokens, teacher_logits, temperature=1.0, weights=None):
    """(losses, gradient of their sum with respect to the logits) of `distillation_loss` from one pass over the logits, for
    steps that know the weights of their rows beforehand: `logits.backward(gradient)` goes on from there.  The
    gradient has the logits' shape and type; the rows of padded logits' gradient are padded too."""
    _check_derivatives(logits, teacher_logits, weights)
    return _distillation(logits, teacher_tokens, teacher_logits, float(temperature), weights, True, True)


def matmul_and_split_qkv(x, weight, bias, num_heads):
    """x [B, L, h] @ weight [h, 3h] + bias, returned as q, k, v [B, num_heads, L, h/num_heads],
    each contiguous; the GEMM's store does the head split."""
    if x.requires_grad:
        _no_gradient("matmul_and_split_qkv")
        x = x.detach()
    batch_size, seqlen, _ = x.shape
    assert x.is_contiguous()
    assert weight.is_contiguous()
    assert x.shape[2] == weight.shape[0]
    hidden_size = weight.shape[1]
    assert hidden_size % 3 == 0, hidden_size
    hidden_size = hidden_size // 3
    assert hidden_size % num_heads == 0, (hidden_size, num_heads)
    head_size = hidden_size // num_heads
    if bias is not None:
        assert bias.is_contiguous()
        assert weight.shape[1] == bias.shape[0]
    dev = _on_gpu(x, weight, bias)
    code = _dtype_code(x, "matmul_and_split_qkv")
    if weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise TypeError("matmul_and_split_qkv: x, weight and bias must share a dtype")
    if head_size % 8 != 0 and isinstance(weight, PackedWeight):
        raise NotImplementedError("matmul_and_split_qkv: packed weights need head_size % 8 == 0")
    if head_size % 8 != 0:
        # the scatter epilogue stores 8-element groups; other head sizes take the plain GEMM
        y = fused_ffn(x, weight, bias=bias)
        q, k, v = y.split(hidden_size, dim=2)
        return tuple(t.view(batch_size, seqlen, num_heads, head_size).transpose(1, 2).contiguous()
                     for t in (q, k, v))
    shape = (batch_size, num_heads, seqlen, head_size)
    q = x.new_empty(shape)
    k = torch.empty_like(q)
    v = torch.empty_like(q)
    lib = _lib.load()
    M, K, N = batch_size * seqlen, x.shape[2], 3 * hidden_size
    wl = _wlayout(weight, _lib.GPTMI_W_KN)
    ws, ws_bytes = _linear_workspace(lib, M, N, K, code, wl, x)
    _call(dev, "matmul_and_split_qkv", lib.gptmi_linear_qkv, x.data_ptr(), weight.data_ptr(),
          _ptr(bias), q.data_ptr(), k.data_ptr(), v.data_ptr(), batch_size, seqlen, num_heads,
          head_size, K, wl, _ptr(ws), ws_bytes, code)
    return q, k, v


def layer_norm_linear_supported(x, weight):
    """True where `layer_norm_ffn` / `layer_norm_matmul_and_split_qkv` take these operands: fp16,
    a packed weight image, a row width the kernel's LDS panel holds."""
    if not isinstance(weight, PackedWeight) or x.dtype != torch.float16:
        return False
    H = x.shape[-1]
    return bool(_lib.load().gptmi_layernorm_linear_supported(x.numel() // H, H, _lib.GPTMI_F16))


def _check_layer_norm_linear(x, ln_weight, ln_bias, weight, bias, what):
    assert x.is_contiguous() and ln_weight.is_contiguous() and ln_bias.is_contiguous()
    assert ln_weight.shape == ln_bias.shape == (x.shape[-1],)
    assert x.shape[-1] == weight.shape[0]
    if not isinstance(weight, PackedWeight):
        raise NotImplementedError(f"{what}: takes the packed image of the weight (pack_weight)")
    if not (x.dtype == ln_weight.dtype == ln_bias.dtype == weight.dtype == torch.float16):
        raise NotImplementedError(f"{what}: fp16 operands only")
    if bias is not None:
        assert bias.is_contiguous() and bias.shape == (weight.shape[1],)
        if bias.dtype != x.dtype:
            raise TypeError(f"{what}: bias is {bias.dtype} but x is {x.dtype}")
    return _on_gpu(x, ln_weight, ln_bias, weight, bias)


def layer_norm_ffn(x, ln_weight, ln_bias, weight, bias=None, add_gelu=False, then=None):
    """gelu?(fused_layer_norm(x, ln_weight, ln_bias) @ weight + bias) in one launch: the
    LayerNorm runs in the GEMM's operand prologue (the fusion marked as to do in the reference,
    kernels.py:132-133) and gives the bits of fused_layer_norm followed by fused_ffn.  Meant for
    few rows; `weight` is a `pack_weight` image, fp16 only (NotImplementedError otherwise, and
    for row widths `layer_norm_linear_supported` turns down).

    then=(weight2, bias2), with add_gelu and bias: the MLP's second product behind it in the same
    call -- the result is x + that @ weight2 + bias2 (fused_ffn with x as the residual, same bits)."""
    if x.requires_grad:
        _no_gradient("layer_norm_ffn")
        x = x.detach()
    if then is not None:
        assert add_gelu and bias is not None
        return mlp_block(x, ln_weight, ln_bias, weight, bias, *then, layer_norm_in_gemm=True)
    dev = _check_layer_norm_linear(x, ln_weight, ln_bias, weight, bias, "layer_norm_ffn")
    K, N = weight.shape
    M = x.numel() // K
    z = x.new_empty((*x.shape[:-1], N))
    _call(dev, "layer_norm_ffn", _lib.load().gptmi_layernorm_linear, x.data_ptr(),
          ln_weight.data_ptr(), ln_bias.data_ptr(), 1e-5, weight.data_ptr(), _ptr(bias),
          z.data_ptr(), M, N, K, 1 if add_gelu else 0, _lib.GPTMI_F16)
    return z


def layer_norm_matmul_and_split_qkv(x, ln_weight, ln_bias, weight, bias, num_heads):
    """matmul_and_split_qkv(fused_layer_norm(x, ln_weight, ln_bias), weight, bias, num_heads) in
    one launch, same bits; see `layer_norm_ffn`.  x [B, L, h]; head size a multiple of 8."""
    if x.requires_grad:
        _no_gradient("layer_norm_matmul_and_split_qkv")
    dev = _check_layer_norm_linear(x, ln_weight, ln_bias, weight, bias,
                                   "layer_norm_matmul_and_split_qkv")
    batch_size, seqlen, K = x.shape
    hidden_size = weight.shape[1] // 3
    assert weight.shape[1] == 3 * hidden_size and hidden_size % num_heads == 0
    head_size = hidden_size // num_heads
    shape = (batch_size, num_heads, seqlen, head_size)
    q = x.new_empty(shape)
    k = torch.empty_like(q)
    v = torch.empty_like(q)
    _call(dev, "layer_norm_matmul_and_split_qkv", _lib.load().gptmi_layernorm_linear_qkv,
          x.data_ptr(), ln_weight.data_ptr(), ln_bias.data_ptr(), 1e-5, weight.data_ptr(),
          _ptr(bias), q.data_ptr(), k.data_ptr(), v.data_ptr(), batch_size, seqlen, num_heads,
          head_size, K, _lib.GPTMI_F16)
    return q, k, v


def flash_attention_v1(q, k, v, dropout_prob=0.0, *, merged_heads_layout=False):
    """Causal softmax(q k^T / sqrt(d)) v for q, k, v [B, N, L, d] -> [B, N, L, d].

    merged_heads_layout=True (an extension; the default is the reference's behaviour)
    returns the same values as a [B, N, L, d]-shaped view of a [B, L, N, d] buffer, so the
    caller's `.transpose(1, 2).contiguous()` head merge costs no copy.
    """
    if q.requires_grad or k.requires_grad or v.requires_grad:
        _no_gradient("flash_attention_v1")
    assert q.shape[:2] == k.shape[:2]
    assert q.shape[-1] == k.shape[-1]
    assert k.shape == v.shape
    B, N, Lq, H = q.shape
    Lk = k.shape[2]
    assert H in HEAD_SIZES
    assert q.is_contiguous()
    assert k.is_contiguous()
    assert v.is_contiguous()
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("flash_attention_v1: q, k and v must share a dtype")
    dev = _on_gpu(q, k, v)
    code = _dtype_code(q, "flash_attention_v1")
    if merged_heads_layout:
        buf = q.new_empty((B, Lq, N, H))
        layout = _lib.GPTMI_O_BLND
    else:
        buf = torch.empty_like(q)
        layout = _lib.GPTMI_O_BNLD
    _call(dev, "flash_attention_v1", _lib.load().gptmi_flash_attn, q.data_ptr(), k.data_ptr(),
          v.data_ptr(), buf.data_ptr(), B, N, Lq, Lk, H, 1 / math.sqrt(H), float(dropout_prob), 1337,
          layout, code)
    return buf.transpose(1, 2) if merged_heads_layout else buf


def _packed_pitches(q, k, v):
    """(q's, k's and v's row and head pitches, their addresses); NotImplementedError where a head does not start at a multiple
    of 16 bytes."""
    (q_row, q_head, q_one), (k_row, k_head, k_one), (v_row, v_head, v_one) = q.stride(), k.stride(), v.stride()
    assert q_one == k_one == v_one == 1, "the elements of a head must lie side by side"
    if q.shape[0] == 1:  # whatever the pitch of one is
        q_row = k_row = v_row = 0
    if q.shape[1] == 1:
        q_head = 0
    if k.shape[1] == 1:
        k_head = v_head = 0
    q_at, k_at, v_at = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if (q_row | q_head | k_row | k_head | v_row | v_head) & 7 or (q_at | k_at | v_at) & 15:
        raise NotImplementedError("flash_attention_packed: heads must start at multiples of 16 bytes")
    return (q_row, q_head, k_row, k_head, v_row, v_head), (q_at, k_at, v_at)


def _packed_attention(q, k, v, starts, scale, out, with_stats):
    """(out, what the gradients need of each row and what the output's rounding takes or None, the scale)."""
    assert q.dim() == k.dim() == 3 and k.shape == v.shape, (q.shape, k.shape, v.shape)
    T, N, d = q.shape
    G = k.shape[1]
    assert k.shape[0] == T and k.shape[2] == d, (q.shape, k.shape)
    assert N > 0 and G > 0 and N % G == 0, (N, G)
    assert d in HEAD_SIZES
    assert starts.dim() == 1 and starts.shape[0] >= 2 and starts.is_contiguous()
    if not q.dtype == k.dtype == v.dtype:
        raise TypeError("flash_attention_packed: q, k and v must share a dtype")
    if q.dtype != torch.float16:
        _dtype_code(q, "flash_attention_packed")
        raise NotImplementedError("flash_attention_packed: fp16 operands only")
    if starts.dtype != torch.int64:
        raise TypeError(f"flash_attention_packed: starts must be int64, got {starts.dtype}")
    dev = _on_gpu(q, k, v, starts, out)
    pitches, (q_at, k_at, v_at) = _packed_pitches(q, k, v)
    if scale is None:
        scale = d ** -0.5
    if not 1e-20 <= scale <= 1e20:
        raise ValueError(f"flash_attention_packed: scale {scale} is not between 1e-20 and 1e20")
    if out is None:
        out = q.new_empty((T, N, d))
    else:
        q_row, q_head, k_row, k_head, v_row, v_head = pitches
        assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
        at = out.data_ptr()
        if at & 15:
            raise NotImplementedError("flash_attention_packed: out must start at a multiple of 16 bytes")
        end = at + 2 * T * N * d
        for start, size, may in ((q_at, 2 * ((T - 1) * q_row + (N - 1) * q_head + d), q.is_contiguous()),
                                 (k_at, 2 * ((T - 1) * k_row + (G - 1) * k_head + d), False),
                                 (v_at, 2 * ((T - 1) * v_row + (G - 1) * v_head + d), False),
                                 (starts.data_ptr(), 8 * starts.shape[0], False)):
            apart = start + size <= at or end <= start
            assert apart or T == 0 or (may and start == at), "out may be a dense q alone"
    stats, remainder = (q.new_empty((N, T, 2), dtype=torch.float32), torch.empty_like(out)) if with_stats else (None, None)
    if T > 0:
        lib, sizes = _lib.load(), (starts.data_ptr(), starts.shape[0] - 1, T, N, G, d, *pitches, scale, _lib.GPTMI_F16)
        if with_stats:
            _call(dev, "flash_attention_packed", lib.gptmi_flash_attn_packed_train_remainder, q_at, k_at, v_at,
                  out.data_ptr(), stats.data_ptr(), remainder.data_ptr(), *sizes)
        else:
            _call(dev, "flash_attention_packed", lib.gptmi_flash_attn_packed, q_at, k_at, v_at, out.data_ptr(), *sizes)
    return out, stats, remainder, scale


# Elements of a row of the output up to which the gradients read it; beyond, the call has an output only.
_MAX_GRADIENT_ROW = 1 << 24


class _PackedAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, starts, scale):
        if q.dim() == 3 and q.shape[1] * q.shape[2] > _MAX_GRADIENT_ROW:
            return _packed_attention(q, k, v, starts, scale, None, False)[0]
        out, stats, remainder, ctx.scale = _packed_attention(q, k, v, starts, scale, None, True)
        ctx.save_for_backward(q, k, v, out, stats, remainder, starts)
        return out

    @staticmethod
    def backward(ctx, d_out):
        _first_derivative("flash_attention_packed")
        saved = ctx.saved_tensors  # once: each reading unpacks them, which checkpoints allow no second time
        if not saved:
            raise NotImplementedError(f"flash_attention_packed: rows of more than {_MAX_GRADIENT_ROW} elements have no gradient")
        q, k, v, out, stats, remainder, starts = saved
        (T, N, d), G = q.shape, k.shape[1]
        need_q, need_k, need_v = ctx.needs_input_grad[:3]
        dq = q.new_empty((T, N, d)) if need_q else None
        dk, dv = (k.new_empty((T, G, d)) for _ in range(2)) if need_k or need_v else (None, None)
        if T > 0:
            d_out = d_out.contiguous()
            if d_out.data_ptr() & 15:
                d_out = d_out.clone()
            pitches, addresses = _packed_pitches(q, k, v)
            lib = _lib.load()
            nbytes = lib.gptmi_flash_attn_packed_backward_workspace_bytes(starts.shape[0] - 1, T, N, G, d)
            workspace = _workspace(nbytes, q)
            _call(q.get_device(), "flash_attention_packed", lib.gptmi_flash_attn_packed_backward_remainder, *addresses,
                  out.data_ptr(), stats.data_ptr(), remainder.data_ptr(), d_out.data_ptr(), starts.data_ptr(), _ptr(dq),
                  _ptr(dk), _ptr(dv), starts.shape[0] - 1, T, N, G, d, *pitches, ctx.scale, workspace.data_ptr(), nbytes, _lib.GPTMI_F16)
        return dq, dk if need_k else None, dv if need_v else None, None, None


def flash_attention_packed(q, k, v, starts, scale=None, out=None):
    """Causal attention over whole prompts of different lengths, one behind the other without padding, with grouped
    heads: q [T, N, d], k and v [T, G, d], N a multiple of G -> [T, N, d].  Sequence s is the rows starts[s] ..
    starts[s + 1] - 1 (int64 on the GPU, S + 1 of them, not decreasing, from 0 to T; a sequence may be empty), scale
    1 / sqrt(d) if None.

    fp16 (fp32 storage would round q, k and v to it).  A head's d elements lie side by side; rows and heads may be
    views of something larger at 16-byte aligned pitches, such as the columns of a q, k, v product.  Rows that belong to no
    sequence are not read, and of `out` not written (dense, allocated if None; a dense q itself may be it, and it may overlap
    nothing else).

    Gradients flow to q, k and v (dense ones, fp16), backward and once; of rows that belong to no sequence they are 0.  Each
    is one sum in one order: the same step gives the same bits.  A call that may have to form them keeps q, k, v, the output, as
    much again for what its rounding takes, and 8 bytes a row and head.  With `out` given the call is a forward pass only, and
    so it is for rows of more than 2^24 elements (N d), whose backward pass raises NotImplementedError."""
    _no_tangents("flash_attention_packed", q, k, v)
    if (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        if out is None:
            return _PackedAttentionFunction.apply(q, k, v, starts, scale)
        _no_gradient("flash_attention_packed with out")
    return _packed_attention(q, k, v, starts, scale, out, False)[0]


class DropoutMask:
    """Bits of the dropout mask that `fused_ffn` (offset m * N + n) and `flash_attention_v1` (offset
    query * Lk + key) draw for probability p: both count flat indices from 0 under one seed, so the
    mask of the largest matrix serves all of them.  `bits` offsets are held."""

    __slots__ = ("data", "bits", "p", "device")

    def __init__(self, data, bits, p):
        self.data, self.bits, self.p, self.device = data, bits, p, data.device

    def serves(self, x, bits, p):
        return self.p == p and bits <= self.bits and self.data.get_device() == x.get_device()


def dropout_mask(bits, p, like):
    """DropoutMask of `bits` offsets (at most 2^32) for 0 < p < 1 on the GPU of `like`."""
    dev = _on_gpu(like)
    lib = _lib.load()
    buf = like.new_empty(lib.gptmi_dropout_mask_bytes(bits), dtype=torch.uint8)
    _call(dev, "dropout_mask", lib.gptmi_dropout_mask, buf.data_ptr(), bits, float(p), 1337)
    return DropoutMask(buf, bits, p)


def _keep_args(keep, x, dropout_prob, what):
    if keep is None:
        return None, 0
    if dropout_prob != keep.p or keep.data.get_device() != x.get_device():
        raise ValueError(f"{what}: the dropout mask is for p = {keep.p} on {keep.device}")
    return keep.data.data_ptr(), keep.bits


# Head sizes of the attention kernels (the reference's set, kernels.py:490).
HEAD_SIZES = frozenset((16, 32, 64, 128, 256))


def block_supported(x, width):
    """True where `attention_block` / `mlp_block` take rows of this width."""
    return width % 64 == 0 and width <= 8192 and x.dtype in _DTYPES


def _block_layout(first, second, what):
    packed = isinstance(first, PackedWeight)
    if packed != isinstance(second, PackedWeight):
        raise TypeError(f"{what}: both weights packed or neither")
    return _lib.GPTMI_W_PACKED if packed else _lib.GPTMI_W_KN


def _in_gemm_code(layer_norm_in_gemm):
    return -1 if layer_norm_in_gemm is None else 1 if layer_norm_in_gemm else 0


def attention_block(x, ln_weight, ln_bias, qkv_weight, qkv_bias, proj_weight, proj_bias, num_heads,
                    dropout_prob=0.0, normed=None, layer_norm_in_gemm=False, keep=None):
    """x + dropout(proj(attention(qkv(LayerNorm(x))))) for x [B, L, h]: the operators of an attention
    block (gpt.py:39-60) behind one call of the library, with their bits in fp16 (fp32: up to the fp16
    rounding of the projection's operands).  `normed`: LayerNorm(x), if the caller has it; layer_norm_in_gemm: as in `layer_norm_matmul_and_split_qkv`
    (False: fp32 blocks of few rows with packed weights all the same; None: in no case); keep: a
    `dropout_mask` for dropout_prob of at least max(x.numel(), L * L) offsets, read instead of
    generating the masks here."""
    if x.requires_grad or normed is not None and normed.requires_grad:
        _no_gradient("attention_block")
    B, L, h = x.shape
    dtype = x.dtype
    assert ln_weight.shape[0] == ln_bias.shape[0] == proj_bias.shape[0] == h
    assert qkv_bias.shape[0] == 3 * h
    dev = _on_gpu(x, ln_weight, ln_bias, qkv_weight, qkv_bias, proj_weight, proj_bias, normed)
    assert x.is_contiguous() and (normed is None or normed.is_contiguous() and normed.shape == x.shape)
    assert ln_weight.is_contiguous() and ln_bias.is_contiguous()
    assert qkv_bias.is_contiguous() and proj_bias.is_contiguous()
    assert qkv_weight.is_contiguous() and proj_weight.is_contiguous()
    assert tuple(qkv_weight.shape) == (h, 3 * h) and tuple(proj_weight.shape) == (h, h)
    assert h % num_heads == 0 and h // num_heads in HEAD_SIZES
    if not (dtype == ln_weight.dtype == ln_bias.dtype == qkv_weight.dtype == qkv_bias.dtype ==
            proj_weight.dtype == proj_bias.dtype and (normed is None or normed.dtype == dtype)):
        raise TypeError("attention_block: x and the parameters must share a dtype")
    code = _dtype_code(x, "attention_block")
    layout = _block_layout(qkv_weight, proj_weight, "attention_block")
    d = h // num_heads
    lib = _lib.load()
    nbytes = lib.gptmi_attention_block_workspace_bytes(B, L, num_heads, d, layout)
    ws = _workspace(nbytes, x)
    out = torch.empty_like(x)
    _call(dev, "attention_block", lib.gptmi_attention_block, x.data_ptr(), _ptr(normed),
          ln_weight.data_ptr(), ln_bias.data_ptr(), 1e-5, qkv_weight.data_ptr(), qkv_bias.data_ptr(),
          proj_weight.data_ptr(), proj_bias.data_ptr(), out.data_ptr(), B, L, num_heads, d,
          float(dropout_prob), 1337, *_keep_args(keep, x, dropout_prob, "attention_block"),
          _in_gemm_code(layer_norm_in_gemm), layout, _ptr(ws), nbytes, code)
    return out


def mlp_block(x, ln_weight, ln_bias, weight1, bias1, weight2, bias2, dropout_prob=0.0,
              layer_norm_in_gemm=False, keep=None):
    """x + dropout(W2 . dropout(gelu(W1 . LayerNorm(x)))): the operators of an MLP block
    (gpt.py:91-111) behind one call of the library, with their bits; layer_norm_in_gemm: as in
    `layer_norm_ffn` and `attention_block`; keep: as in `attention_block`, of at least (rows of x) * max(inner, h) offsets."""
    if x.requires_grad:
        _no_gradient("mlp_block")
    h = x.shape[-1]
    dtype = x.dtype
    inner = weight1.shape[1]
    assert ln_weight.shape[0] == ln_bias.shape[0] == bias2.shape[0] == h and bias1.shape[0] == inner
    dev = _on_gpu(x, ln_weight, ln_bias, weight1, bias1, weight2, bias2)
    assert x.is_contiguous() and ln_weight.is_contiguous() and ln_bias.is_contiguous()
    assert weight1.is_contiguous() and weight2.is_contiguous()
    assert bias1.is_contiguous() and bias2.is_contiguous()
    assert weight1.shape[0] == h and tuple(weight2.shape) == (inner, h)
    if not (dtype == ln_weight.dtype == ln_bias.dtype == weight1.dtype == bias1.dtype ==
            weight2.dtype == bias2.dtype):
        raise TypeError("mlp_block: x and the parameters must share a dtype")
    code = _dtype_code(x, "mlp_block")
    layout = _block_layout(weight1, weight2, "mlp_block")
    M = x.numel() // h
    lib = _lib.load()
    nbytes = lib.gptmi_mlp_block_workspace_bytes(M, h, inner, layout)
    ws = _workspace(nbytes, x)
    out = torch.empty_like(x)
    _call(dev, "mlp_block", lib.gptmi_mlp_block, x.data_ptr(), ln_weight.data_ptr(),
          ln_bias.data_ptr(), 1e-5, weight1.data_ptr(), bias1.data_ptr(), weight2.data_ptr(),
          bias2.data_ptr(), out.data_ptr(), M, h, inner, float(dropout_prob), 1337,
          *_keep_args(keep, x, dropout_prob, "mlp_block"), _in_gemm_code(layer_norm_in_gemm), layout,
          _ptr(ws), nbytes, code)
    return out


def blocks_workspace(x, num_heads, inner):
    """(scratch that serves `block_layers` for x and these sizes, its bytes)."""
    B, L, h = x.shape
    nbytes = _lib.load().gptmi_blocks_workspace_bytes(B, L, num_heads, h // num_heads, inner,
                                                      _dtype_code(x, "block_layers"))
    return _workspace(nbytes, x), nbytes


def block_layers(x, pointers, num_heads, inner, normed=None, layer_norm_in_gemm=False, out=None, workspace=None):
    """`attention_block` then `mlp_block` for each of some layers of a model in one call of the library, packed
    weights, no dropout; same launches, same bits.  pointers: 12 device addresses a layer, as gptmi_blocks
    lists them, of tensors that the caller has checked and keeps (`FusedGPT.forward` does).  out: where the
    result goes, x itself included; workspace: `blocks_workspace`, if the caller has it."""
    if x.requires_grad:
        _no_gradient("block_layers")
    B, L, h = x.shape
    dev = _on_gpu(x, normed, out)
    code = _dtype_code(x, "block_layers")
    assert x.is_contiguous() and (normed is None or normed.is_contiguous() and normed.shape == x.shape)
    assert out is None or out.is_contiguous() and out.shape == x.shape and out.dtype == x.dtype
    assert len(pointers) % 12 == 0 and h % num_heads == 0
    ws, nbytes = workspace or blocks_workspace(x, num_heads, inner)
    if out is None:
        out = torch.empty_like(x)
    table = array.array("Q", pointers)
    _call(dev, "block_layers", _lib.load().gptmi_blocks, x.data_ptr(), _ptr(normed), table.buffer_info()[0],
          len(pointers) // 12, 1e-5, out.data_ptr(), B, L, num_heads, h // num_heads, inner,
          _in_gemm_code(layer_norm_in_gemm), _ptr(ws), nbytes, code)
    return out


def blocks_forward(x, pointers, num_heads, inner, normed=None, layer_norm_in_gemm=False, workspace=None):
    """`block_layers` for a model's layers, or for those that are left of them."""
    return block_layers(x, pointers, num_heads, inner, normed=normed, layer_norm_in_gemm=layer_norm_in_gemm,
                        workspace=workspace)
