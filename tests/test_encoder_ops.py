"""The operators as the package uses them: the encoder with ops="hip" against stock ops, and training steps of it with the
AdamW optimizers; the trainers' options."""
import subprocess
import sys
import os

import pytest
import torch

import artemis_amd
import ops_reference as ref
from artemis_amd.model import ArTEMIS
from artemis_amd.model.encoder import SepSTSBasicLayer, SepSTSEncoder

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"


def layer(ops, dim=32, heads=2, dtype=torch.float32):
    torch.manual_seed(3)
    m = SepSTSBasicLayer(dim, 2, heads, (1, 8, 8), (4, 1, 1))
    for blk in m.blocks:
        blk.ops = blk.norm1.ops = blk.norm2.ops = ops
        for attn in (blk.depth_attn, blk.point_attn):
            torch.nn.init.normal_(attn.relative_position_bias_table, std=0.5)
            torch.nn.init.normal_(attn.qkv.weight, std=dim ** -0.5)
            torch.nn.init.normal_(attn.qkv.bias)
    return m.to(DEV).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(16, 16), (20, 27), (8, 24), (5, 24)])
def test_layer_against_stock_ops_in_64_bits(size):
    """Two blocks (plain and shifted windows, maps padded up to window multiples, a map smaller than a window) against
    the same modules in 64 bits: gradients of input and of all parameters.  A block is some 20 operations deep, each of
    relative rounding sqrt(sum of 32..128 terms) u at most: 2e-5 of the largest element is two orders above that."""
    x = torch.randn(2, 32, 4, *size, generator=torch.Generator().manual_seed(1))
    gy = torch.randn(2, 32, 4, *size, generator=torch.Generator().manual_seed(2))
    results = []
    for ops, dtype in (("hip", torch.float32), ("torch", torch.float64)):
        m = layer(ops, dtype=dtype)
        t = x.to(DEV).to(dtype).requires_grad_(True)
        y = m(t)
        grads = torch.autograd.grad(y, [t, *m.parameters()], gy.to(DEV).to(dtype))
        results.append([("y", y), ("x", grads[0]), *zip((n for n, _ in m.named_parameters()), grads[1:])])
    for (name, got), (_, want) in zip(*results):
        assert got.dtype == torch.float32
        scale = float(want.abs().max())
        # the key bias moves all scores of a row alike: its gradient is 0 but for rounding; qkv's scale counts there
        assert float((got.double() - want).abs().max()) <= 2e-5 * max(scale, 1e-3), name


@pytest.mark.gpu
def test_layer_under_autocast():
    """bf16 products and attention: against fp32, half a step of bf16 (2^-9 of the value) for each of some 30 roundings on the way,
    16 times that for the sums in between."""
    x = torch.randn(1, 32, 4, 16, 16, generator=torch.Generator().manual_seed(1)).to(DEV)
    m = layer("hip")
    want = m(x)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = m(x)
    got.float().sum().backward()
    assert float((got.float() - want).norm() / want.norm()) < 30 * 2.0 ** -9
    assert all(p.grad is not None and p.grad.isfinite().all() for p in m.parameters())


@pytest.mark.gpu
def test_model_interpolates_alike():
    """The whole model at 96 x 160 (its levels are padded, shifted, and smaller than a window at the coarsest)."""
    torch.manual_seed(1)
    stock = ArTEMIS().to(DEV).eval()
    hip = ArTEMIS(encoder_ops="hip").to(DEV).eval()
    hip.load_state_dict(stock.state_dict())
    assert list(hip.state_dict()) == list(stock.state_dict())
    g = torch.Generator().manual_seed(2)
    frames = [torch.rand(1, 3, 96, 160, generator=g).to(DEV) for _ in range(4)]
    a, b = stock.interpolate(frames, [0.25, 0.5]), hip.interpolate(frames, [0.25, 0.5])
    assert float((a - b).abs().max()) <= 1e-4 * float(a.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
def test_training_steps_run(optimizer):
    """Three steps of the model trainer with this package's operators throughout; every parameter with a gradient moves, by at
    most a few times lr (a step of AdamW is no longer than about lr / sqrt(1 - b2) at first)."""
    from artemis_amd.train import ModelTrainer, synthetic_frames
    tr = ModelTrainer(torch.device(DEV), lr=1e-3, encoder_ops="hip", optimizer=optimizer)
    before = [p.detach().clone() for p in tr.module.parameters()]
    for i in range(3):
        assert tr.step(synthetic_frames(1, (64, 64), i, torch.device(DEV))).isfinite()
    moved = 0
    for p, q in zip(tr.module.parameters(), before):
        assert p.isfinite().all()
        d = float((p - q).abs().max())
        assert d <= 3 * (1e-3 * 10 + 1e-5 * float(q.abs().max())) + 1e-6
        moved += d > 0
    assert moved > 0.9 * len(before)
    bits = {"adamw": 9, "adamw8": 2.1}[optimizer]
    held = sum(t.numel() * t.element_size() for s in tr.optimizer.state.values() for t in s.values() if torch.is_tensor(t))
    assert held <= bits * sum(p.numel() for p in before) + 16 * len(before)


@pytest.mark.gpu
def test_command_line():
    r = subprocess.run([sys.executable, "-m", "artemis_amd.train", "--device", "hip:0", "--model", "artemis", "--steps", "2",
                        "--batch", "1", "--size", "64", "--encoder_ops", "hip", "--optimizer", "adamw8",
                        "--cudnn_benchmark", "0"], cwd=ROOT, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert len([ln for ln in r.stdout.splitlines() if ln.startswith("step ")]) == 2


def test_defaults_and_refusals():
    from artemis_amd.main import get_args
    from artemis_amd.train import make_optimizer
    args = get_args([])
    assert args.encoder_ops == "torch" and args.optimizer == "adamax"
    p = [torch.nn.Parameter(torch.zeros(3))]
    assert isinstance(make_optimizer("adamax", p, 1e-3, (0.9, 0.999), 0.0, 1), torch.optim.Adamax)
    with pytest.raises(ValueError):
        make_optimizer("sgd", p, 1e-3, (0.9, 0.999), 0.0, 1)
    with pytest.raises(ValueError):
        SepSTSEncoder([512, 256, 128, 64], 4, [(1, 8, 8)] * 4, [2, 4, 8, 16], ops="cuda")
    # on the CPU the package's operators raise, as the synthesis op does
    enc = SepSTSBasicLayer(32, 1, 2, (1, 8, 8), (4, 1, 1))
    enc.blocks[0].norm1.ops = "hip"
    with pytest.raises(NotImplementedError):
        enc(torch.randn(1, 32, 4, 8, 8))


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["norm", "attention"])
def test_a_capture_beside_an_eager_graph_is_refused(op):
    """With an eager graph of the same leaves alive, torch would tie the capture to the default stream."""
    g = torch.Generator().manual_seed(31)
    if op == "norm":
        x, w = torch.randn(8, 64, generator=g).cuda(), torch.randn(64, generator=g).cuda()
        call = artemis_amd.layer_norm
    else:
        x, w = torch.randn(1, 1, 8, 8, 96, generator=g).cuda(), torch.randn(225, 1, generator=g).cuda()

        def call(a, b):
            return artemis_amd.window_attention(a, b, (1, 8, 8), 1)
    x, w = x.requires_grad_(True), w.requires_grad_(True)

    def step():
        out = call(x, w)
        return (out, *torch.autograd.grad(out, (x, w), torch.ones_like(out)))

    want = [t.detach().clone() for t in step()]
    alive = call(x, w)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="being captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)
        again = step()
        torch.cuda.synchronize()
        assert torch.equal(again[1], want[1])
        del again
