"""AdamW over more tensors than a launch takes (90, with 8-bit moments 59), with sizes next to a workgroup's share of 1024
elements: every tensor against the formulas."""
import pytest
import torch

import artemis_amd
import ops_reference as ref

DEV = "cuda:0"
LR, BETAS, EPS, DECAY, SEED = 3e-3, (0.9, 0.999), 1e-8, 0.05, 5
# 270: three launches of 90, empty tensors among them (which take no place), five of 59
SIZES = [1023, 1024, 1025, 2047, 2048, 2049, 1, 0, 255, 256, 257] + [3 + 7 * k for k in range(268)]


def data(dtype):
    g = torch.Generator().manual_seed(83)
    p = [(0.1 * torch.randn(n, generator=g)).to(dtype) for n in SIZES]
    grad = [(0.01 * torch.randn(n, generator=g)).to(dtype) for n in SIZES]
    return p, grad, g


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_32_bits(dtype):
    p, grad, g = data(dtype)
    m = [0.001 * torch.randn(n, generator=g) for n in SIZES]
    v = [1e-5 * torch.randn(n, generator=g).square() for n in SIZES]
    dev = [[t.to(DEV) for t in ts] for ts in (p, grad, m, v)]
    artemis_amd.adamw_step(*dev, 7, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY)
    for i in range(len(SIZES)):
        want = ref.adamw(p[i], grad[i], m[i], v[i], 7, LR, BETAS, EPS, DECAY)
        for got, (value, bound), name in zip((dev[0][i], dev[2][i], dev[3][i]), want, ("p", "m", "v")):
            ref.assert_within(got, value, bound, f"{name}[{i}]")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_8_bits(dtype):
    """Bit for bit, two steps; the rounding's random numbers go by places that count through all launches."""
    p, grad, _ = data(dtype)
    groups = [(n + 255) // 256 for n in SIZES]
    state = [[torch.zeros(k, dtype=t) for k in (groups if t == torch.int32 else SIZES)]
             for t in (torch.uint8, torch.int32, torch.uint8, torch.int32)]
    dev = [[t.to(DEV) for t in ts] for ts in (p, grad, *state)]
    for step in (1, 2):
        artemis_amd.adamw_step_8bit(*dev, step, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, seed=SEED)
    place = 0
    for i, n in enumerate(SIZES):
        mine = [p[i], *(s[i] for s in state)]
        for step in (1, 2) if n else ():
            mine = list(ref.adamw8(mine[0], grad[i], *mine[1:], step, place, SEED, LR, BETAS, EPS, DECAY))[:5]
        place += groups[i]
        for got, want, name in zip((dev[0][i], *(d[i] for d in dev[2:])), mine, ("p", "m", "m base", "v", "v base")):
            assert torch.equal(got.cpu(), want), (name, i)
