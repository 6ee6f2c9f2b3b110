"""artemis_amd.window_attention against the 64-bit definition: window sizes from one token to thousands, head sizes,
types, shifts, labels with padding and empty rows, and its refusals."""
import math

import pytest
import torch

import artemis_amd
import ops_reference as ref

DEV = "cuda:0"
INF = math.inf


def data(shape, window, heads, hd, dtype, seed, table=True):
    g = torch.Generator().manual_seed(seed)
    entries = (2 * window[0] - 1) * (2 * window[1] - 1) * (2 * window[2] - 1)
    C = heads * hd
    return (torch.randn(*shape, 3 * C, generator=g).to(dtype),
            0.5 * torch.randn(entries, heads, generator=g) if table else None,
            torch.randn(*shape, C, generator=g).to(dtype))


def run(qkv, table, window, heads, dout, labels=None, **kw):
    q = qkv.to(DEV).requires_grad_(True)
    t = None if table is None else table.to(DEV).requires_grad_(True)
    labels = None if labels is None else labels.to(DEV)
    out = artemis_amd.window_attention(q, t, window, heads, labels=labels, **kw)
    grads = torch.autograd.grad(out, [q] if t is None else [q, t], dout.to(DEV))
    with torch.no_grad():
        alone = artemis_amd.window_attention(q, t, window, heads, labels=labels, **kw)
    torch.cuda.synchronize()
    assert torch.allclose(out, alone, rtol=0, atol=0, equal_nan=True)
    return out, list(grads)


def check(qkv, table, window, heads, dout, labels=None, **kw):
    out, grads = run(qkv, table, window, heads, dout, labels, **kw)
    assert out.dtype == qkv.dtype and grads[0].dtype == qkv.dtype
    want = ref.window_attention(qkv, table, window, heads, labels=labels, dout=dout, **kw)
    ref.assert_within(out, *want["out"], "out")
    ref.assert_within(grads[0], *want["dqkv"], "dqkv")
    if table is not None:
        ref.assert_within(grads[1], *want["dtable"], "dtable")
    return out, grads


# (B, D, H, W), window: one token; a few that share 16 slots; sizes next to 16, 32, 64; several key tiles
SHAPES = [
    ((2, 1, 3, 5), (1, 1, 1)), ((2, 4, 3, 7), (4, 1, 1)), ((1, 2, 9, 6), (1, 3, 1)), ((1, 3, 5, 4), (3, 5, 1)),
    ((2, 2, 4, 12), (1, 4, 4)), ((1, 1, 17, 2), (1, 17, 1)), ((1, 2, 8, 8), (2, 4, 4)), ((1, 1, 6, 22), (1, 3, 11)),
    ((2, 4, 16, 24), (1, 8, 8)), ((1, 3, 21, 3), (3, 7, 3)), ((1, 1, 13, 10), (1, 13, 5)), ((1, 4, 8, 16), (4, 8, 8)),
    ((2, 2, 9, 14), (2, 9, 7)), ((1, 1, 129, 1), (1, 129, 1)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,window", SHAPES)
def test_against_64_bits(shape, window, dtype):
    shift = tuple(w // 2 if n > w else 0 for n, w in zip(shape[1:], window))
    qkv, table, dout = data(shape, window, 2, 32, dtype, sum(shape))
    check(qkv, table, window, 2, dout, shift=shift)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hd", [4, 8, 16, 20, 40, 64, 68, 96, 128])
@pytest.mark.parametrize("shape,window", [((2, 4, 2, 3), (4, 1, 1)), ((1, 2, 6, 10), (1, 6, 5)), ((1, 1, 16, 7), (1, 8, 7)),
                                          ((1, 1, 10, 9), (1, 10, 9))])
def test_head_sizes(shape, window, hd, dtype):
    heads = 3
    qkv, table, dout = data(shape, window, heads, hd, dtype, hd)
    check(qkv, table, window, heads, dout)


@pytest.mark.gpu
@pytest.mark.parametrize("outside", [-100.0, -INF, -1.5, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("shape,window", [((2, 2, 8, 12), (1, 4, 4)), ((2, 1, 16, 16), (1, 8, 8)), ((2, 2, 18, 20), (2, 9, 5))])
def test_regions(shape, window, outside):
    """Shift and labels together, a map of labels for each of the batch; padding that leaves whole windows and rows empty."""
    B, D, H, W = shape
    g = torch.Generator().manual_seed(3)
    labels = torch.randint(0, 3, (B, D, H, W), generator=g, dtype=torch.int32)
    labels[0, :, : window[1]] = -1                     # whole windows, cut by the shift
    labels[-1, :, :, -2:] = -(2 ** 31)
    labels[-1, 0, 0, 0] = 2 ** 31 - 1
    qkv, table, dout = data(shape, window, 2, 32, torch.float32, 5)
    shift = (0, window[1] // 2, window[2] // 2)
    out, (dqkv, _) = check(qkv, table, window, 2, dout, labels, shift=shift, outside=outside)
    pad = (labels < 0).to(DEV)
    assert (out[pad] == 0).all() and (dqkv[pad] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("window", [(1, 8, 8), (4, 1, 1), (2, 8, 8)])
def test_padding_is_not_read(window):
    """NaN and infinities in padding reach no other token, its output or its gradient."""
    shape = (1, 4, 8, 16)
    qkv, table, dout = data(shape, window, 2, 32, torch.float32, 7)
    labels = torch.zeros(shape[1:], dtype=torch.int32)
    labels[:, 6:] = -1
    labels[3] = -7
    clean = run(qkv, table, window, 2, dout, labels)
    pad = (labels < 0)[None]
    qkv[pad] = float("nan")
    qkv[:, 3, 0, 0] = INF
    dout[pad] = float("nan")
    dirty = run(qkv, table, window, 2, dout, labels)
    for a, b in zip([clean[0], *clean[1]], [dirty[0], *dirty[1]]):
        assert torch.equal(a, b) and a.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("part", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("window", [(1, 8, 8), (4, 1, 1), (1, 2, 2), (3, 1, 1), (2, 4, 4), (4, 8, 8)])
def test_what_is_not_finite_stays_in_its_window(window, part, dtype):
    """Also where windows share a block of 16 slots."""
    shape = (2, 12, 16, 16)
    qkv, table, dout = data(shape, window, 2, 32, dtype, 9)
    clean, (clean_grad, _) = run(qkv, table, window, 2, dout)
    at = (1, 5, 9, 3)
    if part == "dout":
        dout[at] = float("nan")
    else:
        qkv[at][64 * "qkv".index(part):][:64] = float("inf") if part == "v" else float("nan")
    out, (dqkv, _) = run(qkv, table, window, 2, dout)
    inside = torch.zeros(shape, dtype=torch.bool)
    inside[(1, *(slice(p // w * w, p // w * w + w) for p, w in zip(at[1:], window)))] = True
    inside = inside.to(DEV)
    assert torch.equal(out[~inside], clean[~inside]) and torch.equal(dqkv[~inside], clean_grad[~inside])
    assert not dqkv[inside].isfinite().all() and (part == "dout" or not out[inside].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, 1.0, -0.25, 12.0])
@pytest.mark.parametrize("window", [(1, 4, 4), (1, 8, 8), (1, 16, 8)])
def test_scales(window, scale):
    """Also scores of +- hundreds: one key takes all, and exp2 of the rest underflows."""
    shape = (1, 1, 16, 16)
    qkv, table, dout = data(shape, window, 2, 16, torch.float32, 11)
    check(qkv, table, window, 2, dout, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [(1, 8, 8), (1, 16, 16)])
def test_without_a_table_and_many_windows(window):
    shape = (3, 2, 32, 48)
    qkv, _, dout = data(shape, window, 1, 16, torch.bfloat16, 13, table=False)
    check(qkv, None, window, 1, dout, shift=(0, 3, 5))


@pytest.mark.gpu
def test_more_tiles_than_workgroups():
    """A workgroup meets several tiles: the table's gradient adds over them."""
    shape, window = (2, 4, 192, 192), (4, 1, 1)
    qkv, table, dout = data(shape, window, 2, 4, torch.float32, 15)
    check(qkv, table, window, 2, dout)
    shape, window = (1, 1, 256, 320), (1, 8, 8)
    qkv, table, dout = data(shape, window, 1, 4, torch.float32, 17)
    check(qkv, table, window, 1, dout, shift=(0, 4, 4))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape,window,heads", [((2, 1, 55, 44), (1, 11, 11), 2), ((3, 6, 21, 10), (3, 7, 5), 1)])
def test_many_windows_that_64_tokens_do_not_tile(shape, window, heads, dtype):
    """The table's gradient is summed over shares of the windows."""
    qkv, table, dout = data(shape, window, heads, 16, dtype, 71)
    check(qkv, table, window, heads, dout, shift=(0, 3, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape,window,heads", [((2, 2, 32, 32), (1, 8, 16), 2), ((3, 8, 8, 16), (4, 8, 8), 1)])
def test_many_windows_that_64_tokens_tile(shape, window, heads, dtype):
    """Likewise, by distances of tiles."""
    qkv, table, dout = data(shape, window, heads, 16, dtype, 73)
    check(qkv, table, window, heads, dout, shift=(0, 3, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_the_longest_window(dtype):
    shape = window = (4, 32, 32)
    qkv, table, dout = data((1, *shape), window, 1, 8, dtype, 19)
    labels = torch.zeros(shape, dtype=torch.int32)
    labels[2:] = 1
    labels[:, 31, :16] = -1
    check(qkv, table, window, 1, dout, labels, outside=-INF)


@pytest.mark.gpu
def test_gradient_against_differences():
    """Along one direction, in fp32: f = sum(out dout) at +-t; off by O(t^2) and by the outputs' rounding over t."""
    shape, window = (1, 2, 4, 4), (2, 4, 4)
    qkv, table, dout = data(shape, window, 2, 8, torch.float32, 21)
    g = torch.Generator().manual_seed(2)
    dx, dt = torch.randn(qkv.shape, generator=g), torch.randn(table.shape, generator=g)
    _, (gx, gt) = run(qkv, table, window, 2, dout)
    got = float((gx.double().cpu() * dx).sum() + (gt.double().cpu() * dt).sum())
    t = 2.0 ** -8

    def f(s):  # both in 64 bits, from the definition: what the kernel's gradient is a derivative of
        return float((ref.window_attention((qkv.double() + s * dx), table.double() + s * dt, window, 2)["out"][0] *
                      dout.double()).sum())

    quotient = (8 * (f(t) - f(-t)) - (f(2 * t) - f(-2 * t))) / (12 * t)      # off by f^(5) t^4 / 30
    want = ref.window_attention(qkv, table, window, 2, dout=dout)
    allowed = float((want["dqkv"][1] * dx.abs()).sum() + (want["dtable"][1] * dt.abs()).sum())
    # a fifth derivative of up to 10^4 times the first's scale
    allowed += 1e4 * t ** 4 / 30 * float((want["dqkv"][0] * dx).abs().sum())
    assert abs(got - quotient) <= allowed, (got, quotient, allowed)


@pytest.mark.gpu
def test_same_bits_on_another_stream_unaligned_and_with_an_expanded_gradient():
    shape, window = (2, 4, 16, 16), (1, 8, 8)
    qkv, table, _ = data(shape, window, 2, 32, torch.float32, 23)
    ones = torch.ones(*shape, 64)
    first = run(qkv, table, window, 2, ones, shift=(0, 4, 4))
    flat = torch.empty(qkv.numel() + 1, device=DEV)
    flat[1:] = qkv.reshape(-1).to(DEV)
    view = flat[1:].view(qkv.shape).requires_grad_(True)
    t = table.to(DEV).requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = artemis_amd.window_attention(view, t, window, 2, shift=(0, 4, 4))
        grads = torch.autograd.grad(out.sum(), (view, t))
    side.synchronize()
    for a, b in zip([first[0], *first[1]], [out, *grads]):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [(1, 8, 8), (4, 8, 8)])
def test_forward_and_backward_replay_from_a_graph(window):
    shape = (1, 4, 16, 16)
    x, table, dout = (t.to(DEV) for t in data(shape, window, 2, 32, torch.bfloat16, 25))
    x, table = x.requires_grad_(True), table.requires_grad_(True)

    def step():
        out = artemis_amd.window_attention(x, table, window, 2, shift=(0, 4, 4))
        return (out, *torch.autograd.grad(out, (x, table), dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2, 3):
        nx, nt, nd = data(shape, window, 2, 32, torch.bfloat16, 200 + seed)
        with torch.no_grad():
            x.copy_(nx), table.copy_(nt), dout.copy_(nd)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in captured]
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(got, eager):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [(1, 8, 8), (2, 8, 8)])
def test_an_empty_batch(window):
    q = torch.empty(0, 2, 8, 8, 96, device=DEV, requires_grad=True)
    t = torch.ones((2 * window[0] - 1) * 225, 1, device=DEV, requires_grad=True)
    out = artemis_amd.window_attention(q, t, window, 1)
    dq, dt = torch.autograd.grad(out, (q, t), torch.empty_like(out))
    assert out.shape == (0, 2, 8, 8, 32) and dq.shape == q.shape and torch.equal(dt, torch.zeros_like(dt))


def test_refusals():
    qkv = torch.randn(1, 2, 8, 8, 96)
    table = torch.zeros(225, 1)

    def call(q=qkv, t=table, window=(1, 8, 8), heads=1, **kw):
        return artemis_amd.window_attention(q, t, window, heads, **kw)

    with pytest.raises(NotImplementedError):
        call()
    for error, kw in [
            (TypeError, dict(q=qkv.double())), (ValueError, dict(q=qkv[0])), (ValueError, dict(heads=0)),
            (ValueError, dict(heads=5)), (ValueError, dict(heads=16)),                       # head_dim 2
            (ValueError, dict(q=torch.randn(1, 2, 8, 8, 3 * 132))), (ValueError, dict(window=(1, 8))),
            (ValueError, dict(window=(1, 0, 8))), (ValueError, dict(window=(1, 5, 8))),
            (ValueError, dict(q=torch.randn(1, 1, 65, 64, 12), t=None, window=(1, 65, 64))),  # 4160 tokens
            (ValueError, dict(shift=(0, 8, 0))), (ValueError, dict(shift=(0, -1, 0))), (ValueError, dict(shift=(0, 1))),
            (ValueError, dict(t=torch.zeros(224, 1))), (TypeError, dict(t=table.double())),
            (ValueError, dict(outside=1.0)), (ValueError, dict(outside=math.nan)), (ValueError, dict(scale=INF)),
            (TypeError, dict(labels=torch.zeros(2, 8, 8))), (ValueError, dict(labels=torch.zeros(8, 8, dtype=torch.int32))),
            (AssertionError, dict(q=qkv.transpose(2, 3))),
            (AssertionError, dict(labels=torch.zeros(2, 8, 8, dtype=torch.int32).transpose(1, 2)))]:
        with pytest.raises(error):
            call(**kw)
