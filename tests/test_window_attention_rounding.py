"""artemis_amd.window_attention in 16 bits where roundings add up or values leave the type's range: keys and values far from
zero, gradients so small or so large that dS = P (dP - delta) lies outside fp16's normal numbers, keys that hardly any
query looks at.  Windows are whole maps; the bounds are worst cases of what the kernels round, and hold no measured
number."""
import pytest
import torch

import artemis_amd
import ops_reference as ref

DEV = "cuda:0"
U = ref.U
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])


def definition(q, k, v, do, bias=None):
    """{name: (value, bound)} for (B, heads, n, hd) tensors of a 16-bit type, in 64 bits on the CPU."""
    dtype = q.dtype
    h, f16 = ref.half_step(dtype), dtype == torch.float16
    # A step of P: fp16's subnormal one where the row's largest is 2^15.  A step of dS: where the largest of its row or column
    # met so far is 2^10 or more.  Half of each.  (bf16's lie 100 binades lower.)
    p_step, ds_step = (2.0 ** -40, 2.0 ** -35) if f16 else (0.0, 0.0)
    end_step = ref.smallest_half_step(dtype)
    q, k, v, do = (t.double() for t in (q, k, v, do))
    n, hd = q.shape[-2:]
    scale = hd ** -0.5
    bias = torch.zeros(1, 1, n, n, dtype=torch.float64) if bias is None else bias.double()
    S = scale * q @ k.transpose(-1, -2) + bias
    P = torch.softmax(S, -1)
    out, dP = P @ v, do @ v.transpose(-1, -2)
    delta = (P * dP).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    PT, dST = P.transpose(-1, -2), dS.transpose(-1, -2)
    # fp32: a score is a sum of hd products, scaled, with the bias added, times log2 e; P is off by its score's error, by the
    # sum's (n terms) and by exp2's
    mag = scale * q.abs() @ k.abs().transpose(-1, -2)
    eS = (hd + 4) * U * mag + 8 * U * (1 + mag + bias.abs())
    eP = eS + (P * eS).sum(-1, keepdim=True) + (n + 8) * U                              # relative
    wide = (n + 8) * U                                                                 # sums over tokens
    e_out = (P * (eP + h + wide) + p_step) @ v.abs()
    G = do.abs() @ v.abs().transpose(-1, -2)
    PG = (P * G).sum(-1, keepdim=True)
    # delta is the sum of P dP over the very P that dS is made of: what is relative to all of a row's P moves both alike
    e_delta = (P * eP * dP.abs()).sum(-1, keepdim=True) + (P * eP).sum(-1, keepdim=True) * PG + (n + hd + 8) * U * PG
    e_dS = P * (eP * (dP - delta).abs() + hd * U * G + e_delta + 4 * U * (G + PG))
    if n > 64:
        # dQ: dS is rounded beside a delta that is off by `near` (from the rounded output), which is then taken back out
        # with the sum of P K: left is the rounding of what was off
        near = h * (out.abs() * do.abs()).sum(-1, keepdim=True) + (e_out * do.abs()).sum(-1, keepdim=True) + (hd + 8) * U * PG
    else:
        near = torch.zeros_like(delta)
    A = dS.abs() + P * near
    e_dq = (e_dS + (h + 2 * wide) * A + ds_step * A.amax(-1, keepdim=True)) @ k.abs()
    e_dq = e_dq + near * ((P * (h + 2 * wide) + (2.0 ** -25 if f16 else 0.0)) @ k.abs())
    # dK: by keys (in short windows it was stored by queries before)
    steps = ds_step * (dS.abs().amax(-2, keepdim=True) + dS.abs().amax(-1, keepdim=True))
    e_dk = (e_dS + (h + wide) * dS.abs() + steps).transpose(-1, -2) @ q.abs()
    e_dv = (P * (eP + h + wide) + p_step).transpose(-1, -2) @ do.abs()
    res = {"out": (out, e_out), "dq": (scale * dS @ k, scale * e_dq), "dk": (scale * dST @ q, scale * e_dk), "dv": (PT @ do, e_dv)}
    return {name: (value, e * (1 + h) + h * value.abs() + end_step) for name, (value, e) in res.items()}


def check(q, k, v, do, window, table=None):
    B, heads, n, hd = q.shape
    C = heads * hd

    def on_map(t):  # (B, heads, n, hd) -> (B, D, H, W, C)
        return t.permute(0, 2, 1, 3).reshape(B, *window, C)

    def off_map(t):
        return t.detach().cpu().view(B, n, heads, hd).permute(0, 2, 1, 3)

    qkv = torch.cat([on_map(t) for t in (q, k, v)], -1).to(DEV).requires_grad_(True)
    out = artemis_amd.window_attention(qkv, None if table is None else table.to(DEV), window, heads)
    dqkv, = torch.autograd.grad(out, qkv, on_map(do).to(DEV))
    bias = None if table is None else table[ref.bias_index(window)].permute(2, 0, 1)[None]
    got = dict(zip(("dq", "dk", "dv"), map(off_map, dqkv.split(C, -1))), out=off_map(out))
    for name, (value, bound) in definition(q, k, v, do, bias).items():
        ref.assert_within(got[name], value, bound, name)
    return got


def normal(shape, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(shape, generator=g) for _ in range(4)]


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("offset", [0, 4, 10])
@pytest.mark.parametrize("window,heads", [((1, 8, 8), 2), ((1, 9, 8), 2), ((1, 16, 16), 2), ((1, 11, 30), 1), ((2, 32, 32), 1)])
def test_keys_and_values_far_from_zero(window, heads, offset, dtype):
    """As behind a projection with a bias: an offset of each channel that all keys share moves no gradient of q."""
    q, k, v, do = normal((1, heads, window[0] * window[1] * window[2], 32), 41)
    g = torch.Generator().manual_seed(43)
    k = k + offset * torch.randn(1, heads, 1, 32, generator=g)
    v = v + offset * torch.randn(1, heads, 1, 32, generator=g)
    check(*(t.to(dtype) for t in (0.5 * q, k, v, do)), window)


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("window", [(4, 1, 1), (1, 8, 8), (1, 9, 8), (1, 32, 32), (4, 32, 32)])
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4])
def test_small_gradients(window, size, dtype):
    """dS is about size / n: in fp16 below 2^-14, where steps no longer shrink with the value."""
    q, k, v, do = normal((1, 1, window[0] * window[1] * window[2], 32), 47)
    check(*(t.to(dtype) for t in (q, k, v, size * do)), window)


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("window", [(4, 1, 1), (1, 5, 5), (1, 8, 8), (1, 9, 8), (1, 16, 16)])
def test_large_gradients(window, dtype):
    """dS up to some 2^20, beyond fp16's 65504, where the gradients themselves are not: queries and keys are small."""
    q, k, v, do = normal((2, 2, window[0] * window[1] * window[2], 32), 53)
    got = check(*(t.to(dtype) for t in (q * 2.0 ** -12, k * 2.0 ** -12, v * 512, do * 4096)), window)
    assert all(t.isfinite().all() for t in got.values())


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("window", [(1, 5, 5), (1, 8, 8), (1, 9, 8), (1, 16, 16)])
def test_a_key_that_hardly_any_query_looks_at(window, dtype):
    """Its probabilities, 2^-29 or so, are below fp16's steps; its gradients with a loss scaled by some thousands are not."""
    n = window[0] * window[1] * window[2]
    q, k, v, do = normal((1, 2, n, 32), 59)
    q[..., 0], k[..., 0] = 4.0, 0.0
    k[:, :, 7, 0] = -28.0 + 32 ** -0.5
    v[:, :, 7] *= 1000.0
    got = check(*(t.to(dtype) for t in (0.25 * q, 4 * k, v, 4096 * do)), window)
    assert (got["dv"][:, :, 7] != 0).double().mean() > 0.5
