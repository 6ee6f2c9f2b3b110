"""The operators on tensors of more than 2^32 bytes and 2^31 elements: what lies at the far end against the 64-bit definition,
computed for that end alone."""
import pytest
import torch

import artemis_amd
import ops_reference as ref

DEV = "cuda:0"
ARGS = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)


def spread(shape, dtype, seed):
    """Normal numbers on the GPU, a part at a time: torch's own generator takes 32-bit offsets there."""
    t = torch.empty(shape, dtype=dtype, device=DEV)
    g = torch.Generator(DEV).manual_seed(seed)
    for part in t.view(-1).split(1 << 28):
        part.normal_(generator=g)
    return t


@pytest.fixture(autouse=True)
def _give_memory_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_layer_norm():
    rows, cols = (1 << 25) + 5, 68
    x = spread((rows, cols), torch.bfloat16, 1).requires_grad_(True)
    dy = spread((rows, cols), torch.bfloat16, 2)
    assert x.numel() > 1 << 31
    w, b = torch.linspace(0.5, 1.5, cols), torch.linspace(-1, 1, cols)
    y = artemis_amd.layer_norm(x, w.to(DEV), b.to(DEV))
    dx, = torch.autograd.grad(y, x, dy)
    for part in (slice(0, 40), slice(rows - 40, rows)):
        want = ref.layer_norm(x[part].detach().cpu(), w, b, 1e-5, dy[part].cpu())
        ref.assert_within(y[part], *want["y"], "y")
        ref.assert_within(dx[part], *want["dx"], "dx")


@pytest.mark.gpu
@pytest.mark.parametrize("window", [(1, 8, 8), (1, 2, 2), (1, 16, 16)])
def test_window_attention(window):
    heads, hd, side = 4, 32, 1712
    qkv = spread((2, 1, side, side, 3 * heads * hd), torch.bfloat16, 3).requires_grad_(True)
    dout = spread((2, 1, side, side, heads * hd), torch.bfloat16, 4)
    assert qkv.numel() > 1 << 31
    table = 0.5 * torch.randn((2 * window[1] - 1) * (2 * window[2] - 1), heads, generator=torch.Generator().manual_seed(5))
    out = artemis_amd.window_attention(qkv, table.to(DEV), window, heads)
    dqkv, = torch.autograd.grad(out, qkv, dout)
    n = window[1]
    for batch, h, w in ((0, 0, 0), (1, side - n, side - n)):
        cut = (slice(batch, batch + 1), slice(None), slice(h, h + n), slice(w, w + n))
        want = ref.window_attention(qkv[cut].detach().cpu(), table, window, heads, dout=dout[cut].cpu())
        ref.assert_within(out[cut], *want["out"], "out")
        ref.assert_within(dqkv[cut], *want["dqkv"], "dqkv")


@pytest.mark.gpu
def test_adamw_32_bits():
    n = (1 << 31) + 1027
    p, g = spread((n,), torch.bfloat16, 6), spread((n,), torch.bfloat16, 7)
    m, v = torch.zeros(n, device=DEV), torch.ones(n, device=DEV)
    parts = (slice(0, 2000), slice(n - 2000, n))
    before = [[t[k].cpu() for t in (p, g, m, v)] for k in parts]
    artemis_amd.adamw_step([p], [g], [m], [v], 3, **ARGS)
    for k, old in zip(parts, before):
        want = ref.adamw(*old, 3, ARGS["lr"], ARGS["betas"], ARGS["eps"], ARGS["weight_decay"])
        for got, (value, bound), name in zip((p[k], m[k], v[k]), want, ("p", "m", "v")):
            ref.assert_within(got, value, bound, name)


@pytest.mark.gpu
def test_adamw_8_bits():
    n = (1 << 31) + 1027
    p, g = spread((n,), torch.bfloat16, 8), spread((n,), torch.bfloat16, 9)
    groups = (n + 255) // 256
    s = [torch.zeros(k, dtype=t, device=DEV) for k, t in ((n, torch.uint8), (groups, torch.int32)) * 2]
    first = (1 << 31) // 256                                  # the group that the far part begins with
    parts = ((0, 0, 2048), (first, first * 256, n))
    before = [[t[a:b].cpu() for t in (p, g)] for _, a, b in parts]
    artemis_amd.adamw_step_8bit([p], [g], s[:1], s[1:2], s[2:3], s[3:], 1, seed=11, **ARGS)
    values = artemis_amd.moments_from_8bit(s[:1], s[1:2], signed=True)[0]
    for (group, a, b), old in zip(parts, before):
        count = (b - a + 255) // 256
        zero = [torch.zeros(b - a, dtype=torch.uint8), torch.zeros(count, dtype=torch.int32)]
        want = ref.adamw8(*old, *zero, *zero, 1, group, 11, ARGS["lr"], ARGS["betas"], ARGS["eps"], ARGS["weight_decay"])
        got = (p[a:b], s[0][a:b], s[1][group:group + count], s[2][a:b], s[3][group:group + count])
        for x, value, name in zip(got, want, ("p", "m", "m base", "v", "v base")):
            assert torch.equal(x.cpu(), value), name
        assert torch.equal(values[a:b].cpu(), ref.decode(want[1], want[2], True))
