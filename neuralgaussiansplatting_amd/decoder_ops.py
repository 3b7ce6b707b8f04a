"""Operators over feature rows: what a decoder of the index map's feature map (``rasterizer2``) is built from.

The reference's decoders run on torch's operators (utils/net_utils.py); here a product with everything around it, a norm
and a dropout are one HIP kernel each per direction, for images (millions of narrow rows), wide networks and single
rows.  All three take float32, float16 and bfloat16 tensors on the GPU with any leading dimensions, add and normalise in
32 bits, round each output once, run on the current stream of the tensors' device, and have gradients (first ones:
``create_graph=True`` is refused).  Rows may lie apart (a slice of a wider map is not copied).  Results do not depend on
timing.  The functions come straight from the compiled extension: no Python runs inside a call or its backward pass.
They do not go through torch's dispatcher, so ``torch.autocast`` does not touch them: the tensors' own types decide, and a
call whose tensors' types differ is refused.

``linear(x, weight, bias=None, activation="none", residual=None)``
    ``act(x @ weight.T + bias) + residual``: x [..., in], weight [out, in], bias [out], residual [..., out], all of one
    type.  ``activation`` is "none", "relu", "gelu" (x Phi(x)), "silu" or "sigmoid".  With an activation, the gradients of
    16-bit x and weight are products with dL/dz rounded to their type, which the matrix units take (the bias's gradient sums
    it unrounded); as any float16 gradient, a dL/dz beyond 65504 is infinite.  Where that matters, use float32.

``layer_norm(x, weight=None, bias=None, eps=1e-5)``
    ``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, ``var`` the biased variance; weight and
    bias [width] of x's type or float32.

``dropout(x, p, seed, offset=0, residual=None)``
    ``residual + where(kept, x / (1 - p), 0)``.  Whether an element is kept is a function of (seed, offset, its index),
    so the backward pass stores no mask.  Use another ``offset`` for each dropout of a step and another ``seed`` each
    step.  ``p`` counts in 65536ths, rounded to the nearest.  ``seed`` is a whole number, of which 64 bits count, or one
    int64 on the GPU, read when the kernel runs: a captured graph draws new masks when the tensor is changed between
    replays.  (Changed between a forward pass and its backward pass it would name another mask: that is an error.)
"""
from .diff_gaussian_rasterization._lib import _C

linear = _C.linear
layer_norm = _C.layer_norm
dropout = _C.dropout
