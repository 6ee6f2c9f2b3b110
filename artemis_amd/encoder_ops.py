"""The operators of the Sep-STS encoder (reference: model/sep_sts_layer.py:108-320) as hand-written gfx950
kernels behind the C ABI in ``include/artemis_ops.h``: layer norm, and attention in shifted windows with a
learned relative-position bias and region masks.

    layer_norm(x, weight, bias, eps)                                    -> y, like x
    window_attention(qkv, bias_table, window, num_heads, ...)           -> (B, D, H, W, C)

As for the synthesis op: tensors on a HIP device, contiguous, on torch's current stream; CPU tensors
raise ``NotImplementedError``; no fallback.  fp32, bf16 and fp16; sums, softmax statistics and parameter
gradients are fp32 whatever the type.  No atomics: results are the same bits in every run.  Every call
only enqueues kernels, so it can be captured into a HIP graph.  First derivatives only.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.OPS_F32, torch.bfloat16: _lib.OPS_BF16, torch.float16: _lib.OPS_F16}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _dtype_code(t, what):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _parameter(t, shape, like, what):
    """A parameter as the kernels read it: contiguous fp32 on the input's device.  Another floating type is
    widened by autograd, so that its gradient comes back in that type."""
    if t is None:
        return None
    if not t.is_floating_point() or t.dtype == torch.float64:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{what} must be {shape}, got {tuple(t.shape)}")
    if t.device != like.device:
        raise ValueError(f"{what} is on {t.device}, the input on {like.device}")
    assert (t.is_contiguous() == True)
    return t.float()


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


class FunctionLayerNorm(torch.autograd.Function):
    """``apply(x, weight, bias, eps)``; weight and bias fp32 or None."""

    @staticmethod
    def forward(context, x, weight, bias, eps):
        lib = _lib.load_ops()
        cols = x.size(-1)
        rows = x.numel() // cols if cols else 0
        code = _DTYPES[x.dtype]
        with torch.cuda.device(x.device):
            y = torch.empty_like(x)
            mean = rstd = None
            if any(context.needs_input_grad):
                stats = torch.empty(2, rows, dtype=torch.float32, device=x.device)
                mean, rstd = stats[0], stats[1]
            _lib.check_ops(lib.artemis_ops_layer_norm_forward(
                _ptr(x), _ptr(weight), _ptr(bias), _ptr(y), _ptr(mean), _ptr(rstd), rows, cols, eps, code,
                torch.cuda.current_stream().cuda_stream), "artemis_ops_layer_norm_forward")
        if mean is not None:
            context.save_for_backward(x, weight, mean, rstd)
            context.geom = (rows, cols, code)
        return y

    @staticmethod
    @once_differentiable
    def backward(context, dy):
        x, weight, mean, rstd = context.saved_tensors
        rows, cols, code = context.geom
        need_x, need_w, need_b = context.needs_input_grad[:3]
        lib = _lib.load_ops()
        with torch.cuda.device(x.device):
            dy = dy.contiguous()
            dx = torch.empty_like(x) if need_x else None
            dw = torch.empty(cols, dtype=torch.float32, device=x.device) if need_w else None
            db = torch.empty(cols, dtype=torch.float32, device=x.device) if need_b else None
            nbytes = lib.artemis_ops_layer_norm_workspace_bytes(rows, cols, code) if need_w or need_b else 0
            workspace = _workspace(nbytes, x.device)
            _lib.check_ops(lib.artemis_ops_layer_norm_backward(
                _ptr(x), _ptr(dy), _ptr(weight), _ptr(mean), _ptr(rstd), _ptr(dx), _ptr(dw), _ptr(db), rows, cols,
                code, _ptr(workspace), nbytes, torch.cuda.current_stream().cuda_stream),
                "artemis_ops_layer_norm_backward")
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``torch.nn.functional.layer_norm`` over the last dimension: x (..., C) contiguous fp32, bf16 or fp16;
    weight and bias (C,) or None.  The result has x's type; statistics and the parameters' gradients are
    summed in fp32."""
    _dtype_code(x, "x")
    if x.dim() < 1:
        raise ValueError("x must be (..., C)")
    if not (eps >= 0):
        raise ValueError(f"eps must be >= 0, got {eps}")
    weight = _parameter(weight, (x.size(-1),), x, "weight")
    bias = _parameter(bias, (x.size(-1),), x, "bias")
    assert (x.is_contiguous() == True)
    if not x.is_cuda:
        raise NotImplementedError()
    return FunctionLayerNorm.apply(x, weight, bias, float(eps))


class FunctionWindowAttention(torch.autograd.Function):
    """``apply(qkv, bias_table, labels, desc)``; desc: the fields of ``_lib.WindowDesc`` in order."""

    @staticmethod
    def forward(context, qkv, table, labels, desc):
        lib = _lib.load_ops()
        w = _lib.WindowDesc(*desc)
        with torch.cuda.device(qkv.device):
            out = qkv.new_empty(w.B, w.D, w.H, w.W, w.heads * w.head_dim)
            lse = None
            if any(context.needs_input_grad):
                count = lib.artemis_ops_window_attention_lse_count(ctypes.byref(w))
                if count:
                    lse = torch.empty(count, dtype=torch.float32, device=qkv.device)
            nbytes = lib.artemis_ops_window_attention_workspace_bytes(ctypes.byref(w), 0, 0)
            workspace = _workspace(nbytes, qkv.device)
            _lib.check_ops(lib.artemis_ops_window_attention_forward(
                ctypes.byref(w), _ptr(qkv), _ptr(table), _ptr(labels), _ptr(out), _ptr(lse), _ptr(workspace), nbytes,
                torch.cuda.current_stream().cuda_stream), "artemis_ops_window_attention_forward")
        if any(context.needs_input_grad):
            # short windows: the backward pass computes the softmax again and reads neither
            context.save_for_backward(qkv, table, labels, out if lse is not None else None, lse)
            context.desc = desc
        return out

    @staticmethod
    @once_differentiable
    def backward(context, dout):
        qkv, table, labels, out, lse = context.saved_tensors
        w = _lib.WindowDesc(*context.desc)
        lib = _lib.load_ops()
        with torch.cuda.device(qkv.device):
            dout = _aligned(dout.contiguous())
            dqkv = torch.empty_like(qkv)
            dtable = torch.empty_like(table) if table is not None and context.needs_input_grad[1] else None
            nbytes = lib.artemis_ops_window_attention_workspace_bytes(ctypes.byref(w), 1, int(dtable is not None))
            workspace = _workspace(nbytes, qkv.device)
            _lib.check_ops(lib.artemis_ops_window_attention_backward(
                ctypes.byref(w), _ptr(qkv), _ptr(table), _ptr(labels), _ptr(out), _ptr(lse), _ptr(dout), _ptr(dqkv),
                _ptr(dtable), _ptr(workspace), nbytes, torch.cuda.current_stream().cuda_stream),
                "artemis_ops_window_attention_backward")
        return (dqkv if context.needs_input_grad[0] else None), dtable, None, None


def _aligned(t):
    """The kernels load four elements at once; a view that starts elsewhere is copied."""
    return t if t.data_ptr() % (4 * t.element_size()) == 0 else t.clone()


def _triple(v, what):
    v = tuple(int(n) for n in v)
    if len(v) != 3:
        raise ValueError(f"{what} must be (d, h, w), got {v}")
    return v


def window_attention(qkv, bias_table, window, num_heads, *, shift=(0, 0, 0), labels=None, outside=-100.0,
                     scale=None):
    """Multi-head attention inside (shifted) windows of a (B, D, H, W) map of tokens, with a learned bias that
    depends on the tokens' distance along the three axes -- what model/sep_sts_layer.py:186-219 and :262-300
    compose from a cyclic roll, a window partition, attention with a bias and a mask, and their inverses, as one
    kernel that reads the projection's output where it lies.

    qkv         (B, D, H, W, 3 * num_heads * head_dim) contiguous: what the qkv projection gives for each token
    bias_table  ((2wd-1)(2wh-1)(2ww-1), num_heads) in the reference's order (:134-162), or None
    window      (wd, wh, ww), at most 4096 tokens; D, H, W multiples of it (pad the map first; see ``labels``)
    shift       the window at the origin begins at map position ``shift`` (0 <= shift < window); windows wrap
                around, and tokens from two sides of a wrap are of different regions
    labels      int32 (D, H, W) or (B, D, H, W): tokens of different labels are of different regions (the shots of
                a cut video, say); tokens of a negative label are padding: not attended to, output 0
    outside     added to the scores of tokens of different regions: the reference's -100, or -inf for never
    scale       of q k^T; head_dim ** -0.5 by default
    """
    code = _dtype_code(qkv, "qkv")
    if qkv.dim() != 5:
        raise ValueError(f"qkv must be (B, D, H, W, 3 * C), got {tuple(qkv.shape)}")
    window, shift = _triple(window, "window"), _triple(shift, "shift")
    heads = int(num_heads)
    B, D, H, W, C3 = qkv.shape
    if heads < 1 or C3 % (3 * heads):
        raise ValueError(f"qkv's last dimension {C3} is not 3 * num_heads * head_dim for {heads} heads")
    hd = C3 // (3 * heads)
    if hd % 4 or not 4 <= hd <= 128:
        raise ValueError(f"head_dim {hd} must be a multiple of 4 up to 128")
    if min(window) < 1 or window[0] * window[1] * window[2] > 4096:
        raise ValueError(f"window {window} must hold 1 to 4096 tokens")
    if any(n % w for n, w in zip((D, H, W), window)):
        raise ValueError(f"map {(D, H, W)} is not a multiple of the window {window}")
    if any(not 0 <= s < w for s, w in zip(shift, window)):
        raise ValueError(f"shift {shift} must lie in [0, window) for the window {window}")
    outside, scale = float(outside), hd ** -0.5 if scale is None else float(scale)
    if not outside <= 0:
        raise ValueError(f"outside must be <= 0, got {outside}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    entries = (2 * window[0] - 1) * (2 * window[1] - 1) * (2 * window[2] - 1)
    bias_table = _parameter(bias_table, (entries, heads), qkv, "bias_table")
    maps = 0
    if labels is not None:
        if labels.dtype != torch.int32:
            raise TypeError(f"labels must be int32, got {labels.dtype}")
        if tuple(labels.shape) not in ((D, H, W), (B, D, H, W)):
            raise ValueError(f"labels must be {(D, H, W)} or {(B, D, H, W)}, got {tuple(labels.shape)}")
        if labels.device != qkv.device:
            raise ValueError(f"labels are on {labels.device}, qkv on {qkv.device}")
        assert (labels.is_contiguous() == True)
        maps = B if labels.dim() == 4 and B > 1 else 1
    assert (qkv.is_contiguous() == True)
    if not qkv.is_cuda:
        raise NotImplementedError()
    desc = (B, D, H, W, heads, hd, *window, *shift, maps, code, scale, outside)
    return FunctionWindowAttention.apply(_aligned(qkv), bias_table, labels, desc)
