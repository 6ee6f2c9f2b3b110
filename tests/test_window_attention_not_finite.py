"""artemis_amd.window_attention beside infinities and NaN: what the slots that a window leaves empty, and padding, must not
turn them into.  (Windows of 17 to 63 tokens leave slots of their tile empty, longer ones of their last tile.)"""
import math

import pytest
import torch

import artemis_amd
import ops_reference as ref

DEV = "cuda:0"
INF = math.inf
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
WINDOWS = pytest.mark.parametrize("window", [(3, 1, 1), (1, 3, 7), (1, 5, 5), (1, 7, 7), (1, 8, 8), (1, 9, 8), (1, 12, 12),
                                             (1, 16, 16)])


def data(window, dtype, seed, heads=2, hd=32):
    g = torch.Generator().manual_seed(seed)
    shape = (2, window[0], 2 * window[1], window[2])
    qkv = torch.randn(*shape, 3, heads, hd, generator=g).to(dtype)
    entries = (2 * window[0] - 1) * (2 * window[1] - 1) * (2 * window[2] - 1)
    return qkv, 0.5 * torch.randn(entries, heads, generator=g), torch.randn(*shape, heads * hd, generator=g).to(dtype)


def run(qkv, table, window, dout, labels):
    q = qkv.flatten(4).to(DEV).requires_grad_(True)
    t = table.to(DEV).requires_grad_(True)
    out = artemis_amd.window_attention(q, t, window, 2, labels=None if labels is None else labels.to(DEV))
    return (out, *torch.autograd.grad(out, (q, t), dout.to(DEV)))


def check(got, qkv, table, window, dout, labels, but):
    """Against the definition for a finite stand-in, `but` for those elements of dqkv."""
    want = ref.window_attention(qkv.flatten(4), table, window, 2, dout=dout, labels=labels)
    ref.assert_within(got[0], *want["out"], "out")
    value, bound = want["dqkv"]
    dqkv = torch.where(but.flatten(4), value, got[1].detach().double().cpu())
    ref.assert_within(dqkv, value, bound, "dqkv")
    ref.assert_within(got[2], *want["dtable"], "dtable")


def some_padding(window, padded):
    """Every third token of a raster, in each window; the first is not."""
    if not padded:
        return None
    labels = torch.zeros(window[0], 2 * window[1], window[2], dtype=torch.int32)
    labels.view(-1)[2::3] = -1
    return labels


@pytest.mark.gpu
@TYPES
@WINDOWS
@pytest.mark.parametrize("padded", [False, True])
def test_a_key_at_minus_infinity(window, dtype, padded):
    """No query sees it: outputs and gradients are those beside a key at -30000, whose probabilities are 0 too; but for dQ's
    channel, where 0 meets the infinity."""
    qkv, table, dout = data(window, dtype, 67)
    qkv[..., 0, :, 0] = qkv[..., 0, :, 0].abs() + 0.5
    qkv[0, 0, 0, 0, 1, 1, 0] = -INF
    labels = some_padding(window, padded)
    got = run(qkv, table, window, dout, labels)
    qkv[0, 0, 0, 0, 1, 1, 0] = -30000.0
    but = torch.zeros(qkv.shape, dtype=torch.bool)
    but[0, :, :window[1], :, 0, 1, 0] = True
    check(got, qkv, table, window, dout, labels, but)


@pytest.mark.gpu
@TYPES
@WINDOWS
@pytest.mark.parametrize("padded", [False, True])
def test_a_query_that_sees_nothing(window, dtype, padded):
    """All its scores are -inf: its output is 0, with empty slots or without, and the others' gradients are those
    without it; but for dK's channel, where 0 meets the infinity."""
    qkv, table, dout = data(window, dtype, 71)
    qkv[..., 1, :, 0] = -qkv[..., 1, :, 0].abs() - 0.5
    qkv[0, 0, 0, 0, 0, 1, 0] = INF
    labels = some_padding(window, padded)
    got = run(qkv, table, window, dout, labels)
    assert (got[0][0, 0, 0, 0, 32:] == 0).all()
    # without it: a query of zeros, whose gradient is 0
    qkv[0, 0, 0, 0, 0, 1], dout[0, 0, 0, 0, 32:] = 0, 0
    but = torch.zeros(qkv.shape, dtype=torch.bool)
    but[0, :, :window[1], :, 1, 1, 0] = True
    want = ref.window_attention(qkv.flatten(4), table, window, 2, labels=labels)["out"][0]
    got[0].data[0, 0, 0, 0, 32:] = want[0, 0, 0, 0, 32:].to(got[0])
    check(got, qkv, table, window, dout, labels, but)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("window", [(3, 1, 1), (1, 5, 5), (1, 8, 8), (1, 9, 8)])
@pytest.mark.parametrize("part", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("value", [INF, math.nan])
def test_padding_beside_what_is_not_finite(window, dtype, part, value):
    """Its output and gradients are 0 all the same."""
    qkv, table, dout = data(window, dtype, 73)
    if part == "dout":
        dout[0, 0, 0, 0] = value
    else:
        qkv[0, 0, 0, 0, "qkv".index(part)] = value
    labels = some_padding(window, True)
    out, dqkv, _ = run(qkv, table, window, dout, labels)
    pad = (labels < 0).to(DEV).expand(2, *labels.shape)
    assert (out[pad] == 0).all() and (dqkv[pad] == 0).all()
    assert not dqkv[0].isfinite().all()
