"""The sizes that include/artemis_ops.h gives as limits, on both sides of each, by the host's checks alone."""
import ctypes
import os
import re

import pytest

from artemis_amd import _lib, build


def error():
    return _lib.load_ops().artemis_ops_last_error().decode()


def test_the_header_says_so():
    text = re.sub(r"\s*\n \* +", " ", open(os.path.join(build.INCLUDE, "artemis_ops.h")).read())
    for limit in ("rows below 2^31, cols below 2^30", "B*D*H*W below 2^31; windows * heads below 2^30 for n <= 64",
                  "windows * heads * ceil(n / 64) below 2^24", "at most 2^33 elements", "at most 2^32 places"):
        assert limit in text, limit


@pytest.mark.parametrize("rows,cols,fits", [
    ((1 << 31) - 1, 8, True), (1 << 31, 8, False), (4, (1 << 30) - 1, True), (4, 1 << 30, False)])
def test_layer_norm(rows, cols, fits):
    lib = _lib.load_ops()
    assert lib.artemis_ops_layer_norm_forward(None, None, None, None, None, None, rows, cols, 1e-5, 0, None) == 1
    assert ("NULL" if fits else "columns") in error()       # what fits gets as far as its pointers
    assert lib.artemis_ops_layer_norm_backward(None, None, None, None, None, 16, None, None, rows, cols, 0, None, 0, None) == 1
    assert ("NULL" if fits else "columns") in error()


@pytest.mark.parametrize("B,H,W,heads,window,fits", [
    (1, 2147483645, 1, 1, (1, 5, 1), True), (1, 1 << 16, 1 << 15, 1, (1, 8, 8), False),          # tokens below 2^31
    ((1 << 20) - 1, 2, 2, 1024, (1, 2, 2), True), (1 << 20, 2, 2, 1024, (1, 2, 2), False),        # windows * heads below 2^30
    (4095, 16, 16, 1024, (1, 16, 16), True), (4096, 16, 16, 1024, (1, 16, 16), False),            # times 4 tiles, below 2^24
    (8191, 9, 8, 1024, (1, 9, 8), True), (8192, 9, 8, 1024, (1, 9, 8), False)])                   # times 2
def test_windowed_attention(B, H, W, heads, window, fits):
    lib = _lib.load_ops()
    w = ctypes.byref(_lib.WindowDesc(B, 1, H, W, heads, 4, *window, 0, 0, 0, 0, _lib.OPS_BF16, 0.5, -100.0))
    assert (lib.artemis_ops_window_attention_workspace_bytes(w, 1, 1) > 0) == fits
    assert (lib.artemis_ops_window_attention_lse_count(w) > 0) == (fits and window[1] * window[2] > 64)
    assert lib.artemis_ops_window_attention_forward(w, None, None, None, None, None, None, 0, None) == 1
    assert ("NULL" if fits else "too many") in error()


@pytest.mark.parametrize("bits,count,fits", [(32, 1 << 33, True), (32, (1 << 33) + 1, False), (8, (1 << 32) + 1, False)])
def test_adamw(bits, count, fits):
    one = (_lib.TensorDesc * 1)(_lib.TensorDesc(None if fits else 16, 16, 16, 16, 16, 16, count))
    assert _lib.load_ops().artemis_ops_adamw(one, 1, 0, bits, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 0, None) == 1
    assert ("NULL" if fits else "elements") in error()


def test_the_workspace_that_the_header_names():
    """16 heads of 62 x 62 tokens."""
    w = ctypes.byref(_lib.WindowDesc(1, 1, 62, 62, 16, 32, 1, 62, 62, 0, 0, 0, 0, 0, 0.2, -100.0))
    size = _lib.load_ops().artemis_ops_window_attention_workspace_bytes
    assert 16 * 3844 * 3844 * 4 <= size(w, 1, 1) - size(w, 1, 0) < 16 * 3844 * 3844 * 4 + 64
