"""artemis_amd.layer_norm against the 64-bit definition: types, widths from one column to several thousand (odd ones and
the borders between the kernels' shapes), features far from zero, and its refusals."""
import pytest
import torch

import artemis_amd
import ops_reference as ref

DEV = "cuda:0"


def data(rows, cols, dtype, seed, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * 1.5 + offset * torch.randn(rows, 1, generator=g)).to(dtype)
    return x, 1 + 0.3 * torch.randn(cols, generator=g), 0.3 * torch.randn(cols, generator=g), torch.randn(
        rows, cols, generator=g).to(dtype)


def run(x, w, b, dy, eps=1e-5):
    t = [None if a is None else a.to(DEV).requires_grad_(True) for a in (x, w, b)]
    y = artemis_amd.layer_norm(*t, eps)
    grads = torch.autograd.grad(y, [a for a in t if a is not None], dy.to(DEV))
    torch.cuda.synchronize()
    return y, list(grads)


def check(x, w, b, dy, eps=1e-5):
    y, grads = run(x, w, b, dy, eps)
    want = ref.layer_norm(x, w, b, eps, dy)
    assert y.dtype == x.dtype and grads[0].dtype == x.dtype
    names = ["dx"] + (["dw"] if w is not None else []) + (["db"] if b is not None else [])
    ref.assert_within(y, *want["y"], "y")
    for name, g in zip(names, grads):
        ref.assert_within(g, *want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [
    (1, 1), (3, 2), (1, 7), (5, 8), (33, 32), (257, 64), (1000, 96), (64, 128), (130, 256), (77, 512), (19, 516),
    (65, 1000), (33, 1001), (9, 1024), (7, 2048), (5, 2052), (3, 4096), (5, 4104), (2, 8191), (2, 10000)])
def test_against_64_bits(rows, cols, dtype):
    check(*data(rows, cols, dtype, rows * 10007 + cols))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["none", "weight", "bias"])
def test_parameters_may_be_absent(which):
    x, w, b, dy = data(100, 64, torch.float32, 3)
    check(x, w if which == "weight" else None, b if which == "bias" else None, dy)


@pytest.mark.gpu
def test_many_rows_and_a_large_offset():
    """More rows than workgroups (each adds up several), means 300 times the deviation."""
    x, w, b, dy = data(40000, 64, torch.float32, 5, offset=300.0)
    check(x, w, b, dy)


@pytest.mark.gpu
def test_a_constant_row_and_what_is_not_finite():
    x, w, b, dy = data(8, 64, torch.float32, 7)
    x[2] = 4.0
    clean, _ = run(x, w, b, dy)
    assert torch.equal(clean[2].cpu(), b)             # (x - mean) is exactly 0
    x[5, 3] = float("nan")
    x[6, 1] = float("inf")
    y, (dx, _, _) = run(x, w, b, dy)
    assert y[5].isnan().all() and y[6].isnan().all() and dx[5].isnan().all()
    keep = [0, 1, 2, 3, 4, 7]
    assert torch.equal(y[keep], clean[keep])          # other rows are untouched


@pytest.mark.gpu
def test_unaligned_views_shapes_and_expanded_gradients():
    x, w, b, dy = data(30, 64, torch.float32, 9)
    flat = torch.empty(x.numel() + 1, device=DEV)
    flat[1:] = x.reshape(-1).to(DEV)
    view = flat[1:].view(2, 3, 5, 64).requires_grad_(True)
    assert view.data_ptr() % 16 == 4
    y = artemis_amd.layer_norm(view, w.to(DEV), b.to(DEV))
    assert y.shape == view.shape
    dx, = torch.autograd.grad(y.sum(), view)          # an expanded gradient, no strides
    want = ref.layer_norm(x, w, b, 1e-5, torch.ones_like(dy))
    ref.assert_within(y.view(30, 64), *want["y"], "y")
    ref.assert_within(dx.view(30, 64), *want["dx"], "dx")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cols", [(torch.float32, 1031), (torch.float16, 2051), (torch.bfloat16, 4099)])
def test_rows_over_a_workgroup_at_every_alignment(dtype, cols):
    """More rows than workgroups, each held by all four waves; an odd width in a view that starts off 16 bytes."""
    rows = 1300
    x, w, b, dy = data(rows, cols, dtype, 21)
    flat = torch.empty(x.numel() + 3, dtype=dtype, device=DEV)
    flat[3:] = x.reshape(-1).to(DEV)
    view, wd, bd = flat[3:].view(rows, cols).requires_grad_(True), w.to(DEV).requires_grad_(True), b.to(DEV).requires_grad_(True)
    y = artemis_amd.layer_norm(view, wd, bd)
    grads = torch.autograd.grad(y, (view, wd, bd), dy.to(DEV))
    want = ref.layer_norm(x, w, b, 1e-5, dy)
    for got, name in zip((y, *grads), ("y", "dx", "dw", "db")):
        ref.assert_within(got, *want[name], name)


@pytest.mark.gpu
def test_parameters_of_16_bits_get_gradients_of_their_type():
    x, w, b, dy = data(50, 64, torch.bfloat16, 11)
    w, b = w.bfloat16(), b.bfloat16()
    _, (dx, dw, db) = run(x, w, b, dy)
    want = ref.layer_norm(x, w, b, 1e-5, dy)
    assert dw.dtype == torch.bfloat16
    for got, name in ((dx, "dx"), (dw, "dw"), (db, "db")):
        v, e = want[name]
        ref.assert_within(got, v, e + ref.half_step(torch.bfloat16) * v.abs(), name)


@pytest.mark.gpu
def test_no_rows():
    w = torch.ones(64, device=DEV, requires_grad=True)
    x = torch.empty(0, 64, device=DEV, requires_grad=True)
    y = artemis_amd.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty(0, 64, device=DEV))
    assert y.shape == (0, 64) and dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(dw))


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the kernel's own fp32 output.  With step t the difference quotient of
    f = sum(y dy) is off by the third derivative, O(t^2), and by the output's rounding over t."""
    x, w, b, dy = data(4, 64, torch.float32, 13, offset=0.0)
    t = 2.0 ** -7
    g = torch.Generator().manual_seed(1)
    d = torch.randn(4, 64, generator=g)
    _, (dx, _, _) = run(x, w, b, dy)

    def f(z):
        return (artemis_amd.layer_norm(z.to(DEV), w.to(DEV), b.to(DEV)).double().cpu() * dy.double()).sum()

    got = float((dx.double().cpu() * d.double()).sum())
    quotient = float(f(x + t * d) - f(x - t * d)) / (2 * t)
    # rounding: each of the 512 outputs is off by at most its bound, twice; the cubic term: |f'''| t^2 / 6 with
    # |f'''| <= 40 sum |dy| |d|^3 / sigma^3 for rows of unit-scale features
    e = ref.layer_norm(x, w, b, 1e-5, dy)["y"][1]
    allowed = float((e * dy.abs().double()).sum()) / t + 40 * t * t / 6 * float((dy.abs() * d.abs() ** 3).sum())
    assert abs(got - quotient) <= allowed, (got, quotient, allowed)


@pytest.mark.gpu
def test_same_bits_in_every_run_and_on_another_stream():
    x, w, b, dy = data(20000, 96, torch.bfloat16, 15)
    first = run(x, w, b, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(x, w, b, dy)
    side.synchronize()
    for a, c in zip([first[0], *first[1]], [second[0], *second[1]]):
        assert torch.equal(a, c)


@pytest.mark.gpu
def test_forward_and_backward_replay_from_a_graph():
    x, w, b, dy = (t.to(DEV) for t in data(300, 64, torch.float32, 17))
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))

    def step():
        y = artemis_amd.layer_norm(x, w, b)
        return (y, *torch.autograd.grad(y, (x, w, b), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2, 3):
        nx, _, _, ndy = data(300, 64, torch.float32, 100 + seed)
        with torch.no_grad():
            x.copy_(nx)
            dy.copy_(ndy)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in captured]
        eager = step()
        torch.cuda.synchronize()
        for a, c in zip(got, eager):
            assert torch.equal(a, c)


@pytest.mark.gpu
def test_there_is_no_second_derivative():
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    w = torch.randn(8, device=DEV, requires_grad=True)
    dx, dw = torch.autograd.grad(artemis_amd.layer_norm(x, w).square().sum(), (x, w), create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        (dx.sum() + dw.sum()).backward()
    q = torch.randn(1, 1, 8, 8, 24, device=DEV, requires_grad=True)
    dq, = torch.autograd.grad(artemis_amd.window_attention(q, None, (1, 8, 8), 2).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        dq.sum().backward()


def test_refusals():
    x = torch.randn(4, 8)
    with pytest.raises(NotImplementedError):
        artemis_amd.layer_norm(x)
    with pytest.raises(TypeError):
        artemis_amd.layer_norm(x.double())
    with pytest.raises(TypeError):
        artemis_amd.layer_norm(x, torch.ones(8, dtype=torch.float64))
    with pytest.raises(ValueError):
        artemis_amd.layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError):
        artemis_amd.layer_norm(x, None, torch.ones(1, 8))
    with pytest.raises(ValueError):
        artemis_amd.layer_norm(torch.tensor(1.0))
    with pytest.raises(ValueError):
        artemis_amd.layer_norm(x, eps=-1.0)
    with pytest.raises(AssertionError):
        artemis_amd.layer_norm(x.t())
