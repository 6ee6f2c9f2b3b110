"""The operators of the Sep-STS encoder (reference: model/sep_sts_layer.py:108-320) as hand-written gfx950
kernels behind the C ABI in ``include/artemis_ops.h``: layer norm, and attention in shifted windows with a
learned relative-position bias and region masks.

    layer_norm(x, weight, bias, eps)                                    -> y, like x
    window_attention(qkv, bias_table, window, num_heads, ...)           -> (B, D, H, W, C)

As for the synthesis op: tensors on a HIP device, contiguous (asserted), on torch's current stream; CPU
tensors raise ``NotImplementedError``; no fallback.  fp32, bf16 and fp16; sums, softmax statistics and
parameter gradients are fp32 whatever the type.  In bf16 and fp16 the attention's probabilities, and in the backward pass
dS = P (dP - delta), are rounded to the type as operands of the products with V, dout, Q and K, once each (in fp16 scaled, so
that they lie in its normal range): outputs and gradients are off by about 1.4 times what rounding them alone would be.  No
atomics: results are the same bits in every run.  Every
call only enqueues kernels, so it can be captured into a HIP graph -- a backward pass while no graph of the same
leaves that was made on the default stream is alive (refused).  First derivatives only.  The host side of a
call (checks, memory, autograd) is csrc/ops_torch.cpp.
"""
from __future__ import annotations

from . import _lib


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``torch.nn.functional.layer_norm`` over the last dimension: x (..., C) contiguous fp32, bf16 or fp16;
    weight and bias (C,) or None.  The result has x's type; statistics and the parameters' gradients are
    summed in fp32."""
    return _lib.load_ops_host().layer_norm(x, weight, bias, eps)


def window_attention(qkv, bias_table, window, num_heads, *, shift=(0, 0, 0), labels=None, outside=-100.0,
                     scale=None):
    """Multi-head attention inside (shifted) windows of a (B, D, H, W) map of tokens, with a learned bias that
    depends on the tokens' distance along the three axes -- what model/sep_sts_layer.py:186-219 and :262-300
    compose from a cyclic roll, a window partition, attention with a bias and a mask, and their inverses, as one
    kernel that reads the projection's output where it lies.

    qkv         (B, D, H, W, 3 * num_heads * head_dim) contiguous: what the qkv projection gives for each token;
                head_dim a multiple of 4 up to 128
    bias_table  ((2wd-1)(2wh-1)(2ww-1), num_heads) in the reference's order (:134-162), or None
    window      (wd, wh, ww), at most 4096 tokens; D, H, W multiples of it (pad the map first; see ``labels``)
    shift       the window at the origin begins at map position ``shift`` (0 <= shift < window); windows wrap
                around, and tokens from two sides of a wrap are of different regions
    labels      int32 (D, H, W) or (B, D, H, W): tokens of different labels are of different regions (the shots of
                a cut video, say); tokens of a negative label are padding: not read, not attended to, output 0
    outside     added to the scores of tokens of different regions: the reference's -100, or -inf for never
    scale       of q k^T; head_dim ** -0.5 by default

    Sizes: B * D * H * W below 2^31; windows * heads below 2^30, in windows of more than 64 tokens windows * heads *
    ceil(tokens / 64) below 2^24.  The gradient of bias_table in windows of n > 64 tokens that runs of 64 do not tile
    evenly takes heads * n * n * 4 bytes of memory during the backward pass, times the shares where windows are many and
    short (16 heads of 62 x 62 tokens: 0.95 GB).
    """
    return _lib.load_ops_host().window_attention(qkv, bias_table, window, num_heads, shift, labels, outside, scale)
