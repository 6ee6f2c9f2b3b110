"""Plain 64-bit restatements of layer norm, windowed attention and AdamW, with bounds on what rounding may do to a
32-bit evaluation of them.

u = 2^-24 is half a step of fp32, h = finfo(t).eps / 2 half a step of the output's type.  A sum of n terms
that is added up in chains of length c is off by at most c u times the sum of the terms' magnitudes; the
bounds below use the longest chain that a kernel may have and add the terms up by absolute value, element by
element.  They contain no measured number.
"""
import math

import numpy as np
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest_half_step(dtype):
    """Below 2^-14 the steps of fp16 stay 2^-24 wide (fp32 and bf16: 2^-149 and 2^-133): half of one is what rounding
    may do there, whatever the value."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def assert_within(got, want, bound, what):
    """|got - want| <= bound on every element; infinities and NaN where the reference has them."""
    got = got.detach().double().cpu()
    want, bound = want.detach().double().cpu(), bound.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin), what + ": finite in other places"
    over = (got - want).abs()[fin] - bound.expand_as(want)[fin]
    if over.numel():
        k = int(over.argmax())
        assert float(over[k]) <= 0, (f"{what}: off by {float((got - want).abs()[fin][k]):.3e} at element {k}, "
                                     f"{float(bound.expand_as(want)[fin][k]):.3e} allowed")


# ------------------------------------------------------------------------------------------ layer norm

def layer_norm(x, w, b, eps, dy=None):
    """{name: (value, bound)} in 64 bits for x (rows, C) of any type."""
    rows, C = x.shape
    h = half_step(x.dtype) if x.dtype != torch.float32 else U
    least = smallest_half_step(x.dtype)
    x = x.double()
    w = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    b0 = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    var = xc.square().mean(-1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    xh = xc * r
    chain = C / 8 + 32        # at least 8 lanes share a row, then a tree and a division
    e_mean = chain * U * x.abs().mean(-1, keepdim=True)
    e_xc = e_mean + U * (x.abs() + mean.abs())
    # relative error of rstd: half the relative error of var + eps, and the root and the division
    e_r = 0.5 * (2 * (xc.abs() * e_xc).mean(-1, keepdim=True) + e_mean ** 2 + chain * U * var) / (var + eps) + 4 * U
    e_xh = r * e_xc + xh.abs() * (e_r + 2 * U)
    y = xh * w + b0
    out = {"y": (y, (e_xh * w.abs() + 2 * U * ((xh * w).abs() + b0.abs())) * (1 + h) + h * y.abs() + least)}
    if dy is None:
        return out
    dy = dy.double()
    a = dy * w
    m1, m2 = a.mean(-1, keepdim=True), (a * xh).mean(-1, keepdim=True)
    e_m1 = chain * U * a.abs().mean(-1, keepdim=True) + U * a.abs().mean(-1, keepdim=True)
    e_m2 = (chain + 2) * U * (a * xh).abs().mean(-1, keepdim=True) + (a.abs() * e_xh).mean(-1, keepdim=True)
    dx = r * (a - m1 - xh * m2)
    e = r * (U * a.abs() + e_m1 + xh.abs() * e_m2 + m2.abs() * e_xh + 3 * U * (a.abs() + m1.abs() + (xh * m2).abs()))
    e = e + dx.abs() * (e_r + 2 * U)
    out["dx"] = (dx, e * (1 + h) + h * dx.abs() + least)
    chain = rows + 32
    g = dy.abs()
    out["dw"] = ((dy * xh).sum(0), (g * e_xh).sum(0) + (min(chain, 4096) * U + 2 * U) * (g * xh.abs()).sum(0))
    out["db"] = (dy.sum(0), min(chain, 4096) * U * g.sum(0))
    return out


# ------------------------------------------------------------------------------------------- attention

def bias_index(window):
    axes = torch.stack(torch.meshgrid(*[torch.arange(n) for n in window], indexing="ij")).reshape(3, -1)
    d = axes[:, :, None] - axes[:, None] + torch.tensor([n - 1 for n in window]).view(3, 1, 1)
    return (d[0] * (2 * window[1] - 1) + d[1]) * (2 * window[2] - 1) + d[2]


def _cut(t, window, shift):
    """(B, D, H, W, c) -> (B, windows, n, c)"""
    B, D, H, W, c = t.shape
    wd, wh, ww = window
    t = torch.roll(t, tuple(-s for s in shift), (1, 2, 3))
    t = t.reshape(B, D // wd, wd, H // wh, wh, W // ww, ww, c).permute(0, 1, 3, 5, 2, 4, 6, 7)
    return t.reshape(B, -1, wd * wh * ww, c)


def _paste(t, shape, window, shift):
    B, D, H, W = shape
    wd, wh, ww = window
    t = t.reshape(B, D // wd, H // wh, W // ww, wd, wh, ww, -1).permute(0, 1, 4, 2, 5, 3, 6, 7).reshape(B, D, H, W, -1)
    return torch.roll(t, tuple(shift), (1, 2, 3))


def window_attention(qkv, table, window, heads, shift=(0, 0, 0), labels=None, outside=-100.0, scale=None, dout=None):
    """{name: (value, bound)} in 64 bits, on the CPU."""
    qkv_dtype = qkv.dtype
    t16 = qkv_dtype in (torch.bfloat16, torch.float16)
    h = half_step(qkv_dtype) if t16 else U
    qkv = qkv.detach().double().cpu()
    B, D, H, W, C3 = qkv.shape
    C = C3 // 3
    hd, n = C // heads, window[0] * window[1] * window[2]
    scale = hd ** -0.5 if scale is None else scale
    # regions of the wrapped map
    region = torch.zeros(D, H, W, dtype=torch.long)
    for axis, (size, s) in enumerate(zip((D, H, W), shift)):
        shape = [1, 1, 1]
        shape[axis] = size
        region = region * 2 + (torch.arange(size) < s).long().view(shape)
    region = _cut(region[None, ..., None].double(), window, shift)[..., 0]             # (1, nW, n)
    lab = torch.zeros(1, D, H, W) if labels is None else labels.double().cpu().reshape(-1, D, H, W)
    lab = _cut(lab[..., None].double(), window, shift)[..., 0]                         # (1 | B, nW, n)
    differ = (region[..., :, None] != region[..., None, :]) | (lab[..., :, None] != lab[..., None, :])
    never = (lab[..., :, None] < 0) | (lab[..., None, :] < 0)
    mask = torch.zeros(differ.shape, dtype=torch.float64)
    mask[differ] = outside
    mask[never] = -math.inf
    pad = (lab < 0)[..., None, :, None]                                                # (., nW, 1, n, 1)
    x = _cut(qkv, window, shift).reshape(B, -1, n, 3, heads, hd).permute(3, 0, 1, 4, 2, 5)   # (3, B, nW, h, n, hd)
    q, k, v = (torch.where(pad, torch.zeros((), dtype=torch.float64), t) for t in x)
    bias = torch.zeros(heads, n, n, dtype=torch.float64)
    if table is not None:
        bias = table.detach().double().cpu()[bias_index(window)].permute(2, 0, 1)
    S = scale * q @ k.transpose(-1, -2) + bias + mask[:, :, None]
    dead = (S == -math.inf).all(-1, keepdim=True)
    S0 = torch.where(dead, torch.zeros_like(S), S)
    P = torch.where(dead, torch.zeros_like(S), torch.softmax(S0, -1))
    out = P @ v
    # bounds.  A score is a sum of hd products, scaled, with bias and mask added, times log2 e; its exponential is
    # relatively off by the score's absolute error (and by exp2's own, two steps); the row sum by n u.
    # (scores that the mask moves by `outside`: the rounding of the moved score counts)
    mag = abs(scale) * q.abs() @ k.abs().transpose(-1, -2)
    size = mag + bias.abs() + torch.where(torch.isfinite(mask), mask.abs(), torch.zeros_like(mask))[:, :, None]
    eS = (hd + 4) * U * mag + 8 * U * (1 + size)
    live = torch.where(P > 0, eS, torch.zeros_like(eS))
    eP = live + (P * live).sum(-1, keepdim=True) + (n + 8) * U                          # relative
    # in 16 bits P, dS and (long windows) the fading factors' products are rounded to half a step of the type
    hp = h if t16 else 0.0
    tiny = torch.finfo(torch.float16).smallest_normal * 2.0 ** -10 if qkv_dtype == torch.float16 else 2.0 ** -126  # subnormal steps
    e_out = (P * (eP + hp + (n + 8) * U)) @ v.abs() + tiny * v.abs().sum(-2, keepdim=True)

    def back(t):
        return _paste(t.permute(0, 1, 3, 2, 4).reshape(B, -1, n, C), (B, D, H, W), window, shift)

    res = {"out": (back(out), back(e_out) * (1 + h) + h * back(out).abs() + tiny)}
    if dout is None:
        return res
    do = _cut(dout.detach().double().cpu(), window, shift).reshape(B, -1, n, heads, hd).permute(0, 1, 3, 2, 4)
    do = torch.where(pad, torch.zeros((), dtype=torch.float64), do)
    PT = P.transpose(-1, -2)
    dv = PT @ do
    dP = do @ v.transpose(-1, -2)
    G = do.abs() @ v.abs().transpose(-1, -2)
    delta = (P * dP).sum(-1, keepdim=True)
    PG = (P * G).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    e_delta = (P * eP * dP.abs()).sum(-1, keepdim=True) + (n + hd + 8) * U * PG
    e_dS = P * (eP * (dP - delta).abs() + hd * U * G + e_delta + 4 * U * (G + PG))
    # long windows in 16 bits: dQ is computed with delta from the rounded output
    near = (h * (out.abs() * do.abs()).sum(-1, keepdim=True) + ((P * (eP + hp)) @ v.abs() * do.abs()).sum(-1, keepdim=True)
            + (hd + 8) * U * PG) if n > 64 else torch.zeros_like(delta)
    s = abs(scale)
    dq, dk = scale * dS @ k, scale * dS.transpose(-1, -2) @ q
    e_dq = s * ((e_dS + P * near + (hp + (n + 8) * U) * dS.abs() + tiny) @ k.abs())
    e_dk = s * ((e_dS + (hp + (n + 8) * U) * dS.abs() + tiny).transpose(-1, -2) @ q.abs())
    e_dv = (P * (eP + hp + (n + 8) * U) + tiny).transpose(-1, -2) @ do.abs()
    grads = [(dq, e_dq), (dk, e_dk), (dv, e_dv)]
    val = torch.cat([back(g) for g, _ in grads], -1)
    res["dqkv"] = (val, torch.cat([back(e) for _, e in grads], -1) * (1 + h) + h * val.abs() + tiny)
    if table is not None:
        index = bias_index(window).reshape(-1)

        def fold(t):
            flat = t.sum((0, 1)).reshape(heads, n * n).t()
            return torch.zeros(table.shape, dtype=torch.float64).index_add_(0, index, flat)

        # chains: the windows that a workgroup meets, then its partners, then the pairs of an entry
        terms = min(B * dS.shape[1], 4096) + n + 64
        res["dtable"] = (fold(dS), fold(e_dS) + terms * U * fold(dS.abs()) + 1e-37)
    return res


# ----------------------------------------------------------------------------------------------- AdamW

GROUP = 256


def adamw(p, g, m, v, step, lr, betas, eps, wd):
    """((p, bound), (m, bound), (v, bound)) in 64 bits; the bounds count the roundings of the fp32 formulas."""
    h = half_step(p.dtype) if p.dtype != torch.float32 else U
    least = smallest_half_step(p.dtype)
    p, g, m, v = (t.double() for t in (p, g, m, v))
    b1, b2 = betas
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    # a coefficient's rounding, a product's, the sum's
    e_m = 3 * U * (b1 * m.abs() + (1 - b1) * g.abs()) + 2e-45
    e_v = 4 * U * v1 + 4e-45
    root = torch.sqrt(v1 / (1 - b2 ** step))
    up = lr / (1 - b1 ** step) * m1 / (root + eps)
    # sqrt halves a relative error; a subnormal v has few digits: its absolute error counts
    e_root = torch.where(v1 > 0, torch.sqrt((v1 + e_v) / (1 - b2 ** step)) - root, torch.zeros_like(root))
    e_up = lr / (1 - b1 ** step) * e_m / (root + eps) + up.abs() * (8 * U + e_root / (root + eps))
    new = p * (1 - lr * wd) - up
    return ((new, (3 * U * p.abs() + e_up + U * new.abs()) * (1 + h) + h * new.abs() + least), (m1, e_m), (v1, e_v))


def _bits(x):
    return x.contiguous().view(torch.int32).long()


def _floats(bits):
    return bits.to(torch.int32).view(torch.float32)


def _groups(n):
    return (n + GROUP - 1) // GROUP


def _tops(x):
    """The largest magnitude's bit pattern in each group of 256 of a flat fp32 tensor, for every element's group."""
    n = x.numel()
    padded = torch.zeros(_groups(n) * GROUP, dtype=torch.float32)
    padded[:n] = x.abs()
    return _bits(padded).view(-1, GROUP).amax(1)


def noise(count, group0, step, seed):
    key = (seed * 0x9E3779B1 + step * 0x6A09E667) & 0xFFFFFFFF
    z = (torch.arange(count) + group0 * GROUP + key) & 0xFFFFFFFF
    z = ((z ^ (z >> 16)) * 0x6A09E667) & 0xFFFFFFFF
    z = ((z ^ (z >> 15)) * 0x3B67AE85) & 0xFFFFFFFF
    return z ^ (z >> 16)


def encode(x, random16, signed):
    """8-bit codes and bases of a flat fp32 CPU tensor."""
    most = 127 if signed else 255
    base = ((_tops(x) >> 20) + 1 - most).clamp_min(0)
    each = base.repeat_interleave(GROUP)[:x.numel()]
    a = x.abs()
    code = ((_bits(a) + (random16 << 4)) >> 20) - each
    if signed:
        least = _floats((each + 1) << 20)
        code = torch.where(a < least, (a * 65536.0 > random16.float() * least).long(), code.clamp(max=most))
        code = code + 128 * ((x < 0) & (code > 0)).long()
    else:
        code = torch.where(a > 0, code.clamp(1, most), torch.zeros_like(code))
    return code.to(torch.uint8), base.to(torch.int32)


def decode(codes, bases, signed):
    c = codes.long()
    low = c & 127 if signed else c
    each = bases.long().repeat_interleave(GROUP)[:c.numel()]
    v = _floats(torch.where(low > 0, (low + each) << 20, torch.zeros_like(low)))
    return torch.where(c > 127, -v, v) if signed else v


def adamw8(p, g, mc, mb, vc, vb, step, group0, seed, lr, betas, eps, wd):
    """One flat CPU tensor's step, operation by operation in fp32 as the kernel rounds them: equal bits."""
    (b1, b2), dtype = betas, p.dtype
    p, g = p.float(), g.float()
    m = decode(mc, mb, True) * b1 + g * (1 - b1)
    v = decode(vc, vb, False) * b2 + g * g * (1 - b2)
    p = p * (1 - lr * wd)
    root = torch.from_numpy(np.sqrt(v.numpy()))  # IEEE's; torch's on the CPU is off by a last bit for one value in six
    p = p - m * (lr / (1 - b1 ** step)) / (root * (1 / math.sqrt(1 - b2 ** step)) + eps)
    z = noise(p.numel(), group0, step, seed)
    return (p.to(dtype), *encode(m, z & 0xFFFF, True), *encode(v, z >> 16, False), m, v)
