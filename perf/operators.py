"""What the encoder's operators and the optimizer step are measured on: layer norm, windowed attention with a
relative-position bias and region masks, and the AdamW step over many tensors.

``run`` computes them in their plain form, from elementary torch operations in 32 bits, or -- where ``own`` is true --
through the package's entry points ``artemis_amd.layer_norm``, ``artemis_amd.window_attention``,
``artemis_amd.adamw_step`` and ``artemis_amd.adamw_step_8bit``.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BETAS, EPS, DECAY, LR, SEED = (0.9, 0.999), 1e-8, 1e-2, 2e-4, 103
#: elements that share one exponent base in the 8-bit moments
BLOCK = 256


# ---------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # the coarsest encoder level of one 128 x 128 crop: latency counts
        {"name": "norm small f32", "op": "norm", "dtype": "f32", "rows": 256, "cols": 512, "train": True},
        # the finest encoder level (1/2 of 256 x 256) of 8 crops x 4 frames in training
        {"name": "norm train f32", "op": "norm", "dtype": "f32", "rows": 524288, "cols": 64, "train": True},
        # the 1/8 level of a 1080p window of 4 frames in bf16
        {"name": "norm train bf16", "op": "norm", "dtype": "bf16", "rows": 130560, "cols": 256, "train": True},
        # rows of an odd width, inference
        {"name": "norm odd f16", "op": "norm", "dtype": "f16", "rows": 8191, "cols": 1001, "train": False},
        # coarsest level of one 256 x 256 crop: 16 windows of 64 tokens, 16 heads
        {"name": "attention small f32", "op": "attention", "dtype": "f32", "B": 1, "D": 4, "H": 16, "W": 16, "wd": 1, "wh": 8,
         "ww": 8, "heads": 16, "hd": 32, "sh": 0, "sw": 0, "outside": -100.0, "labels": False, "train": True},
        # finest level of 8 crops in training, a block on shifted windows
        {"name": "attention shifted f32", "op": "attention", "dtype": "f32", "B": 8, "D": 4, "H": 128, "W": 128, "wd": 1, "wh": 8,
         "ww": 8, "heads": 2, "hd": 32, "sh": 4, "sw": 4, "outside": -100.0, "labels": False, "train": True},
        # attention over time: 4 frames at each pixel, the 1/4 level of 8 crops
        {"name": "attention time f32", "op": "attention", "dtype": "f32", "B": 8, "D": 4, "H": 64, "W": 64, "wd": 4, "wh": 1,
         "ww": 1, "heads": 4, "hd": 32, "sh": 0, "sw": 0, "outside": -100.0, "labels": False, "train": True},
        # the 1/4 level of a 1080p window (270 rows padded to 272), interpolation
        {"name": "attention 1080p bf16", "op": "attention", "dtype": "bf16", "B": 1, "D": 4, "H": 272, "W": 480, "wd": 1, "wh": 8,
         "ww": 8, "heads": 4, "hd": 32, "sh": 4, "sw": 4, "outside": -100.0, "labels": False, "train": False},
        # one window over 4 whole 32 x 32 feature maps, with labels (two shots and a padded border), in training
        {"name": "attention long bf16", "op": "attention", "dtype": "bf16", "B": 1, "D": 4, "H": 32, "W": 32, "wd": 4, "wh": 32,
         "ww": 32, "heads": 8, "hd": 32, "sh": 0, "sw": 0, "outside": -math.inf, "labels": True, "train": True},
        # one small sub-network of a synthesis head
        {"name": "adamw small", "op": "adamw", "dtype": "f32", "bits": 32, "tensors": 8, "total": 60000, "step": 1},
        # the whole model's parameters
        {"name": "adamw model", "op": "adamw", "dtype": "f32", "bits": 32, "tensors": 320, "total": 29090528, "step": 1000},
        {"name": "adamw model 8 bit", "op": "adamw", "dtype": "f32", "bits": 8, "tensors": 320, "total": 29090528, "step": 1000},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges: any type, both directions, sizes over the whole range, odd ones among them."""
    op = rng.choice(["norm", "attention", "attention", "adamw"])
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    if op == "norm":
        cols = _log_int(rng, 1, 8192)
        if rng.random() < 0.6:
            cols = max(8, cols // 8 * 8)
        rows = _log_int(rng, 1, max(1, min(524288, 33000000 // cols)))
        return {"op": "norm", "dtype": dtype, "rows": rows, "cols": cols, "train": rng.random() < 0.7}
    if op == "adamw":
        total = _log_int(rng, 1000, 29000000)
        return {"op": "adamw", "dtype": dtype, "bits": rng.choice([32, 8]), "tensors": rng.randint(1, 320), "total": total,
                "step": _log_int(rng, 1, 100000)}
    while True:
        kind = rng.choice(["space", "time", "volume"])
        if kind == "space":
            wd, wh, ww = 1, rng.randint(1, 16), rng.randint(1, 16)
        elif kind == "time":
            wd, wh, ww = rng.randint(1, 32), 1, 1
        else:
            wd, wh, ww = rng.randint(1, 4), _log_int(rng, 1, 32), _log_int(rng, 1, 32)
        n = wd * wh * ww
        heads, hd = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([8, 16, 20, 32, 32, 32, 48, 64, 96, 128])
        # at most the largest listed case's values and products
        most = min(33000000 // (heads * hd), 130000000 // (n * heads))
        if most < n:
            continue
        windows = _log_int(rng, 1, most // n)
        nw = rng.randint(1, max(1, int(math.sqrt(windows))))
        nh = max(1, windows // nw)
        B = rng.randint(1, 4) if nh >= 4 else 1
        nh = max(1, nh // B)
        return {"op": "attention", "dtype": dtype, "B": B, "D": wd, "H": nh * wh, "W": nw * ww, "wd": wd, "wh": wh, "ww": ww,
                "heads": heads, "hd": hd, "sh": rng.randrange(wh) if nh > 1 else 0, "sw": rng.randrange(ww) if nw > 1 else 0,
                "outside": rng.choice([-100.0, -math.inf]), "labels": rng.random() < 0.4, "train": rng.random() < 0.7}


def _sizes(case):
    """Element counts of the tensors of an optimizer case: log-spread, odd ones among them, adding up to about `total`."""
    rng = random.Random(case["tensors"] * 1000003 + case["total"])
    raw = [math.exp(rng.uniform(0.0, 8.0)) for _ in range(case["tensors"])]
    scale = case["total"] / sum(raw)
    return [max(1, int(r * scale)) for r in raw]


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


# --------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = {"case": dict(case)}
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        # features away from zero, as behind a residual sum
        s["x"] = (randn(rows, cols) * 1.5 + 0.5 * randn(rows, 1)).to(dtype).requires_grad_(case["train"])
        s["weight"] = (1 + 0.1 * randn(cols)).requires_grad_(case["train"])
        s["bias"] = (0.1 * randn(cols)).requires_grad_(case["train"])
        s["dy"] = randn(rows, cols).to(dtype) if case["train"] else None
    elif case["op"] == "attention":
        B, D, H, W, C = case["B"], case["D"], case["H"], case["W"], case["heads"] * case["hd"]
        s["qkv"] = randn(B, D, H, W, 3 * C).to(dtype).requires_grad_(case["train"])
        table = (2 * case["wd"] - 1) * (2 * case["wh"] - 1) * (2 * case["ww"] - 1)
        s["table"] = (0.5 * randn(table, case["heads"])).requires_grad_(case["train"])
        s["dout"] = randn(B, D, H, W, C).to(dtype) if case["train"] else None
        s["labels"] = None
        if case["labels"]:
            # two shots in time, and a last row of padding
            lab = torch.zeros(D, H, W, dtype=torch.int32, device=dev)
            lab[D // 2:] = 1
            lab[:, H - 1:, : (W + 1) // 2] = -1
            s["labels"] = lab
    else:
        sizes = _sizes(case)
        starts, at = [], 0
        for n in sizes:
            starts.append(at)
            at += _blocks(n) * BLOCK
        live = torch.zeros(at, device=dev)
        for b, n in zip(starts, sizes):
            live[b:b + n] = 1
        # gradients of very different sizes from tensor to tensor, a few of them zero
        size = torch.repeat_interleave(10 ** (-4 + 3 * torch.rand(len(sizes), generator=g, device=dev)),
                                       torch.tensor([_blocks(n) * BLOCK for n in sizes], device=dev))
        keep = (torch.rand(at, generator=g, device=dev) > 0.01).float()
        s["flat_p"] = (0.05 * randn(at) * live).to(dtype)
        s["flat_g"] = (randn(at) * size * live * keep).to(dtype)
        m = 0.1 * randn(at) * size * live
        v = (randn(at) * size).square() * live * 0.1
        if case["step"] == 1:
            m, v = torch.zeros_like(m), torch.zeros_like(v)

        def views(flat):
            return [flat[b:b + n] for b, n in zip(starts, sizes)]

        s["params"], s["grads"] = views(s["flat_p"]), views(s["flat_g"])
        if case["bits"] == 32:
            s["flat_m"], s["flat_v"] = m, v
            s["m"], s["v"] = views(m), views(v)
        else:
            at_block = [b // BLOCK for b in starts]
            noise = torch.randint(0, 1 << 16, (2, at), generator=g, device=dev)
            s["m_codes"], s["m_bases"] = _encode_signed(m, noise[0])
            s["v_codes"], s["v_bases"] = _encode_positive(v, noise[1])
            s["m_code_list"], s["v_code_list"] = views(s["m_codes"]), views(s["v_codes"])
            s["m_base_list"] = [s["m_bases"][b:b + _blocks(n)] for b, n in zip(at_block, sizes)]
            s["v_base_list"] = [s["v_bases"][b:b + _blocks(n)] for b, n in zip(at_block, sizes)]
    return s


# ----------------------------------------------------------------------------------------------- plain

def _plain_norm(s):
    eps = 1e-5
    x, w, b = s["x"].detach().float(), s["weight"].detach(), s["bias"].detach()
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt(xc.square().mean(-1, keepdim=True) + eps)
    xh = xc * rstd
    y = (xh * w + b).to(s["x"].dtype)
    if s["dy"] is None:
        return {"y": y}
    dy = s["dy"].float()
    dxh = dy * w
    dx = rstd * (dxh - dxh.mean(-1, keepdim=True) - xh * (dxh * xh).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dw": (dy * xh).sum(0), "db": dy.sum(0)}


def _window_positions(case, dev):
    """For each window and token of it: the position in the (D, H, W) map, and which axes the cyclic shift wrapped."""
    D, H, W = case["D"], case["H"], case["W"]
    wd, wh, ww = case["wd"], case["wh"], case["ww"]
    p = torch.arange(D * H * W, device=dev)
    d, h, w = p // (H * W), p // W % H, p % W
    hs, wsft = h + case["sh"], w + case["sw"]
    wrapped = (hs >= H).long() * 2 + (wsft >= W).long()
    place = (d * H + hs % H) * W + wsft % W

    def cut(t):
        return t.view(D // wd, wd, H // wh, wh, W // ww, ww).permute(0, 2, 4, 1, 3, 5).reshape(-1, wd * wh * ww)

    return cut(place), cut(wrapped)


def _bias_index(case, dev):
    wd, wh, ww = case["wd"], case["wh"], case["ww"]
    t = torch.arange(wd * wh * ww, device=dev)
    d, h, w = t // (wh * ww), t // ww % wh, t % ww
    return (((d[:, None] - d[None] + wd - 1) * (2 * wh - 1) + h[:, None] - h[None] + wh - 1) * (2 * ww - 1)
            + w[:, None] - w[None] + ww - 1)


def _plain_attention(s):
    case, qkv = s["case"], s["qkv"].detach()
    dev, dtype = qkv.device, qkv.dtype
    B, D, H, W = qkv.shape[:4]
    h, hd = case["heads"], case["hd"]
    C = h * hd
    place, wrapped = _window_positions(case, dev)
    nw, n = place.shape
    where = place.reshape(-1)
    x = qkv.reshape(B, D * H * W, 3 * C)[:, where].float().view(B * nw, n, 3, h, hd).permute(2, 0, 3, 1, 4).contiguous()
    q, k, v = x[0], x[1], x[2]
    index = _bias_index(case, dev)
    scale = hd ** -0.5
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    score += s["table"].detach()[index].permute(2, 0, 1)
    if case["sh"] or case["sw"] or s["labels"] is not None:
        lab = s["labels"].reshape(-1)[place] if s["labels"] is not None else torch.zeros_like(wrapped)
        differ = (lab[:, :, None] != lab[:, None]) | (wrapped[:, :, None] != wrapped[:, None])
        never = (lab[:, :, None] < 0) | (lab[:, None] < 0)
        mask = torch.zeros(differ.shape, device=dev).masked_fill(differ, case["outside"]).masked_fill(never, -math.inf)
        score.view(B, nw, h, n, n).add_(mask[None, :, None])
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    del score
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    del e
    o = torch.matmul(p, v)

    def back(t):
        """(B * nw, h, n, hd) -> (B, D, H, W, C)"""
        out = torch.empty(B, D * H * W, C, device=dev)
        out[:, where] = t.permute(0, 2, 1, 3).reshape(B, nw * n, C)
        return out.view(B, D, H, W, C).to(dtype)

    out = back(o)
    if s["dout"] is None:
        return {"out": out}
    do = s["dout"].reshape(B, D * H * W, C)[:, where].float().view(B * nw, n, h, hd).permute(0, 2, 1, 3).contiguous()
    dv = torch.matmul(p.transpose(-1, -2), do)
    dp = torch.matmul(do, v.transpose(-1, -2).contiguous())
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    del p, dp
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(-1, -2), q) * scale
    # up to millions of pairs share one entry of the table: summed in 64 bits
    pairs = ds.sum(0, dtype=torch.float64).view(h, n * n).t()
    dtable = torch.zeros(s["table"].shape, dtype=torch.float64, device=dev).index_add_(0, index.reshape(-1), pairs)
    return {"out": out, "dqkv": torch.cat([back(dq), back(dk), back(dv)], -1), "dtable": dtable.float()}


def _bits(x):
    """The bit pattern of positive 32-bit floats, as whole numbers that order as the floats do."""
    return x.contiguous().view(torch.int32).long()


def _floats(bits):
    return bits.to(torch.int32).view(torch.float32)


def _encode_positive(v, noise):
    """Values >= 0 in 8 bits: the top 8 + 3 bits of the 32-bit float, counted up from a base of the block, the rest
    rounded up or down at random (16 bits of `noise`) so that the mean is right.  0 stands for 0 alone."""
    bits = _bits(v)
    base = ((bits.view(-1, BLOCK).amax(1) >> 20) + 1 - 255).clamp_min(0)
    code = ((bits + (noise << 4)) >> 20) - base.repeat_interleave(BLOCK)
    code = torch.where(v > 0, code.clamp(1, 255), torch.zeros_like(code))
    return code.to(torch.uint8), base.to(torch.int32)


def _encode_signed(m, noise):
    """The same with a sign and 7 bits; below the smallest code either that or 0, at random, with the right mean."""
    bits = _bits(m.abs())
    base = ((bits.view(-1, BLOCK).amax(1) >> 20) + 1 - 127).clamp_min(0).repeat_interleave(BLOCK)
    code = (((bits + (noise << 4)) >> 20) - base).clamp(max=127)
    least = _floats((base + 1) << 20)
    small = m.abs() < least
    code = torch.where(small, (m.abs() * 65536.0 > noise.float() * least).long(), code)
    code = code + 128 * ((m < 0) & (code > 0)).long()
    return code.to(torch.uint8), base.view(-1, BLOCK)[:, 0].to(torch.int32)


def _decode_positive(codes, bases):
    c = codes.long()
    return _floats(torch.where(c > 0, (c + bases.long().repeat_interleave(BLOCK)) << 20, torch.zeros_like(c)))


def _decode_signed(codes, bases):
    c = codes.long()
    v = _decode_positive(c & 127, bases)
    return torch.where(c > 127, -v, v)


def _noise(n, step, dev):
    """32 random bits for each element: its place, the step and the seed, mixed by multiplications and shifts."""
    low = 0xFFFFFFFF
    key = (SEED * 0x9E3779B1 + step * 0x6A09E667) & low
    z = (torch.arange(n, device=dev) + key) & low
    z = ((z ^ (z >> 16)) * 0x6A09E667) & low
    z = ((z ^ (z >> 15)) * 0x3B67AE85) & low
    return z ^ (z >> 16)


def _plain_adamw(s):
    case = s["case"]
    (b1, b2), step = BETAS, case["step"]
    p, g = s["flat_p"].float(), s["flat_g"].float()
    if case["bits"] == 32:
        m, v = s["flat_m"], s["flat_v"]
    else:
        m = _decode_signed(s["m_codes"], s["m_bases"])
        v = _decode_positive(s["v_codes"], s["v_bases"])
    m.mul_(b1).add_(g * (1 - b1))
    v.mul_(b2).add_(g * g * (1 - b2))
    p.mul_(1 - LR * DECAY)
    p.sub_(m * (LR / (1 - b1 ** step)) / (torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** step)) + EPS))
    s["flat_p"].copy_(p)
    if case["bits"] == 32:
        return {"p": s["flat_p"], "m": m, "v": v}
    z = _noise(m.numel(), step, m.device)
    codes, bases = _encode_signed(m, z & 0xFFFF)
    s["m_codes"].copy_(codes), s["m_bases"].copy_(bases)
    codes, bases = _encode_positive(v, z >> 16)
    s["v_codes"].copy_(codes), s["v_bases"].copy_(bases)
    return {"p": s["flat_p"], "m": _decode_signed(s["m_codes"], s["m_bases"]),
            "v": _decode_positive(s["v_codes"], s["v_bases"])}


# ------------------------------------------------------------------------------------------------- own

def _own(s):
    import artemis_amd
    case = s["case"]
    if case["op"] == "norm":
        if s["dy"] is None:
            return {"y": artemis_amd.layer_norm(s["x"], s["weight"], s["bias"], 1e-5)}
        y = artemis_amd.layer_norm(s["x"], s["weight"], s["bias"], 1e-5)
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if case["op"] == "attention":
        window, shift = (case["wd"], case["wh"], case["ww"]), (0, case["sh"], case["sw"])
        out = artemis_amd.window_attention(s["qkv"], s["table"], window, case["heads"], shift=shift, labels=s["labels"],
                                           outside=case["outside"])
        if s["dout"] is None:
            return {"out": out}
        dqkv, dtable = torch.autograd.grad(out, (s["qkv"], s["table"]), s["dout"])
        return {"out": out, "dqkv": dqkv, "dtable": dtable}
    if case["bits"] == 32:
        artemis_amd.adamw_step(s["params"], s["grads"], s["m"], s["v"], case["step"], lr=LR, betas=BETAS, eps=EPS,
                               weight_decay=DECAY)
        return {"p": s["flat_p"], "m": s["flat_m"], "v": s["flat_v"]}
    artemis_amd.adamw_step_8bit(s["params"], s["grads"], s["m_code_list"], s["m_base_list"], s["v_code_list"], s["v_base_list"],
                                case["step"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, seed=SEED)
    m, = artemis_amd.moments_from_8bit([s["m_codes"]], [s["m_bases"]], signed=True)
    v, = artemis_amd.moments_from_8bit([s["v_codes"]], [s["v_bases"]], signed=False)
    return {"p": s["flat_p"], "m": m, "v": v}


@torch.no_grad()
def _plain(s):
    op = s["case"]["op"]
    return _plain_norm(s) if op == "norm" else _plain_attention(s) if op == "attention" else _plain_adamw(s)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ work

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": n * size * (4 if case["train"] else 2) + 16 * case["cols"], "flops": n * (20 if case["train"] else 8)}
    if case["op"] == "attention":
        tokens, C = case["B"] * case["D"] * case["H"] * case["W"], case["heads"] * case["hd"]
        n = case["wd"] * case["wh"] * case["ww"]
        table = (2 * case["wd"] - 1) * (2 * case["wh"] - 1) * (2 * case["ww"] - 1) * case["heads"] * 4
        if case["train"]:  # qkv, dout in; out, dqkv out; seven products of 2 n hd for each token and head would do less
            return {"bytes": 8 * tokens * C * size + 2 * table, "flops": 14 * tokens * n * C}
        return {"bytes": 4 * tokens * C * size + table, "flops": 4 * tokens * n * C}
    n = sum(_sizes(case))
    moments = 16 if case["bits"] == 32 else 4
    # 8-bit moments come back as the values they stand for: read once and written in 32 bits
    return {"bytes": n * (3 * size + moments + (0 if case["bits"] == 32 else 10)), "flops": 15 * n}


# ----------------------------------------------------------------------------------------------- exact

@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    f8 = torch.float64
    if case["op"] == "norm":
        x, w, b = s["x"].to(f8), s["weight"].to(f8), s["bias"].to(f8)
        var, mean = torch.var_mean(x, -1, keepdim=True, unbiased=False)
        r = 1 / torch.sqrt(var + 1e-5)
        y = (x - mean) * r
        if not case["train"]:
            return {"y": y * w + b}
        dy = s["dy"].to(f8)
        a = dy * w
        # the projection onto what mean and variance leave free
        dx = r * (a - a.sum(-1, keepdim=True) / x.shape[1] - y * ((a * y).sum(-1, keepdim=True) / x.shape[1]))
        return {"y": y * w + b, "dx": dx, "dw": (dy * y).sum(0), "db": dy.sum(0)}
    if case["op"] == "adamw":
        g = s["flat_g"].to(f8)
        if case["bits"] == 32:
            m, v = s["flat_m"].to(f8), s["flat_v"].to(f8)
        else:
            def value(code, base):  # exponent and three bits of mantissa by arithmetic
                q = code.to(f8) + base.to(f8).repeat_interleave(BLOCK)
                e = torch.floor(q / 8)
                x = torch.where(e > 0, torch.exp2(e.clamp_min(1) - 127) * (1 + (q - 8 * e) / 8), (q - 8 * e) / 8 * 2.0 ** -126)
                return torch.where(code > 0, x, torch.zeros_like(x))
            low = s["m_codes"] % 128
            m = value(low, s["m_bases"]) * torch.where(s["m_codes"] >= 128, -1.0, 1.0)
            v = value(s["v_codes"], s["v_bases"])
        t = case["step"]
        m = BETAS[0] * m + (1 - BETAS[0]) * g
        v = BETAS[1] * v + (1 - BETAS[1]) * g ** 2
        p = s["flat_p"].to(f8) * (1 - LR * DECAY)
        p = p - LR * (m / (1 - BETAS[0] ** t)) / ((v / (1 - BETAS[1] ** t)) ** 0.5 + EPS)
        # the 8-bit moments are rounded at random: no value in 64 bits
        return {"p": p, "m": m, "v": v} if case["bits"] == 32 else {"p": p, "m": None, "v": None}
    # attention, one axis of the map after the other rolled and cut into windows; head by head
    wd, wh, ww, h, hd = case["wd"], case["wh"], case["ww"], case["heads"], case["hd"]
    B, D, H, W = case["B"], case["D"], case["H"], case["W"]
    C, n, dev = h * hd, wd * wh * ww, s["qkv"].device

    def cut(t):  # (B, D, H, W, c) -> (B, windows, n, c)
        t = torch.roll(t, (-case["sh"], -case["sw"]), (2, 3))
        t = t.reshape(t.shape[0], D // wd, wd, H // wh, wh, W // ww, ww, -1).permute(0, 1, 3, 5, 2, 4, 6, 7)
        return t.reshape(t.shape[0], -1, n, t.shape[-1])

    def paste(t):
        t = t.reshape(B, D // wd, H // wh, W // ww, wd, wh, ww, -1).permute(0, 1, 4, 2, 5, 3, 6, 7).reshape(B, D, H, W, -1)
        return torch.roll(t, (case["sh"], case["sw"]), (2, 3))

    # regions: what the roll brought round from the other side is a region of its own on each axis
    rows, cols = torch.arange(H, device=dev) < case["sh"], torch.arange(W, device=dev) < case["sw"]
    region = (rows[:, None].long() * 2 + cols[None].long()).expand(D, H, W)
    lab = torch.zeros(D, H, W, device=dev, dtype=torch.long) if s["labels"] is None else s["labels"].long()
    region, lab = (cut(t[None, ..., None])[0, ..., 0] for t in (region, lab))
    add = torch.zeros(region.shape[0], n, n, dtype=f8, device=dev)
    add[(region[:, :, None] != region[:, None]) | (lab[:, :, None] != lab[:, None])] = case["outside"]
    add[(lab[:, :, None] < 0) | (lab[:, None] < 0)] = -math.inf
    axes = torch.stack(torch.meshgrid(*[torch.arange(k, device=dev) for k in (wd, wh, ww)], indexing="ij")).reshape(3, -1)
    diff = axes[:, :, None] - axes[:, None] + torch.tensor([wd - 1, wh - 1, ww - 1], device=dev).view(3, 1, 1)
    index = (diff[0] * (2 * wh - 1) + diff[1]) * (2 * ww - 1) + diff[2]
    x = cut(s["qkv"].to(f8))
    do = cut(s["dout"].to(f8)) if case["train"] else None
    outs, dqs, dks, dvs, tables = [], [], [], [], []
    for i in range(h):
        q, k, v = (x[..., j * C + i * hd:j * C + (i + 1) * hd].contiguous() for j in range(3))
        a = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(hd) + s["table"][:, i].to(f8)[index] + add
        dead = (a == -math.inf).all(-1, keepdim=True)
        a = torch.where(dead, torch.zeros_like(a), a)
        p = torch.where(dead, torch.zeros_like(a), torch.softmax(a, -1))
        del a
        outs.append(torch.matmul(p, v))
        if case["train"]:
            e = do[..., i * hd:(i + 1) * hd].contiguous()
            dvs.append(torch.matmul(p.transpose(-1, -2).contiguous(), e))
            dp = torch.matmul(e, v.transpose(-1, -2).contiguous())
            dp = p * (dp - (p * dp).sum(-1, keepdim=True))
            dqs.append(torch.matmul(dp, k) / math.sqrt(hd))
            dks.append(torch.matmul(dp.transpose(-1, -2).contiguous(), q) / math.sqrt(hd))
            tables.append(torch.zeros(s["table"].shape[0], dtype=f8, device=dev).index_add_(0, index.reshape(-1),
                                                                                          dp.sum((0, 1)).reshape(-1)))
    out = paste(torch.cat(outs, -1))
    if not case["train"]:
        return {"out": out}
    return {"out": out, "dqkv": paste(torch.cat(dqs + dks + dvs, -1)), "dtable": torch.stack(tables, 1)}
