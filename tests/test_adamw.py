"""The AdamW step over many tensors: 32-bit moments against the 64-bit formulas, 8-bit ones bit for bit against the same
operations on the CPU, what the rounding at random must keep, the optimizer class, and the refusals."""
import math

import pytest
import torch

import artemis_amd
import ops_reference as ref
from artemis_amd.optim import AdamW

DEV = "cuda:0"
ARGS = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)
# one element, the borders of groups (256), shares (4096) and launches (64 tensors), odd ones
SIZES = [1, 2, 3, 4, 5, 255, 256, 257, 1023, 4095, 4096, 4097, 10001, 70000] + [7 + 13 * k for k in range(60)]


def data(sizes, dtype, seed, spread=3):
    g = torch.Generator().manual_seed(seed)
    p, gr, m, v = [], [], [], []
    for n in sizes:
        s = 10 ** float(-spread * torch.rand(1, generator=g))
        p.append((0.1 * torch.randn(n, generator=g)).to(dtype))
        gr.append((s * torch.randn(n, generator=g) * (torch.rand(n, generator=g) > 0.1)).to(dtype))
        m.append(0.1 * s * torch.randn(n, generator=g))
        v.append(0.1 * s * s * torch.randn(n, generator=g).square())
    return p, gr, m, v


def on(ts):
    return [t.to(DEV) for t in ts]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("step", [1, 2, 1000, 10 ** 6])
def test_32_bits_against_64(dtype, step):
    p, g, m, v = data(SIZES, dtype, step)
    if step == 1:
        m, v = [torch.zeros_like(t) for t in m], [torch.zeros_like(t) for t in v]
    dp, dg, dm, dv = on(p), on(g), on(m), on(v)
    versions = [t._version for t in dp]
    artemis_amd.adamw_step(dp, dg, dm, dv, step, **ARGS)
    torch.cuda.synchronize()
    assert all(t._version > k for t, k in zip(dp, versions))     # autograd's saved parameters are out of date
    for i in range(len(p)):
        want = ref.adamw(p[i], g[i], m[i], v[i], step, ARGS["lr"], ARGS["betas"], ARGS["eps"], ARGS["weight_decay"])
        for got, (value, bound), name in zip((dp[i], dm[i], dv[i]), want, ("p", "m", "v")):
            ref.assert_within(got, value, bound, f"{name}[{i}]")
        assert torch.equal(dg[i].cpu(), g[i])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_unaligned_neighbours_and_zeros(bits):
    """Tensors that begin anywhere in a buffer, back to back: nothing beside them is written.  Zero gradients and
    moments with eps > 0 leave the decayed parameter."""
    sizes = [5, 1, 300, 4099, 2]
    total = sum(sizes) + 3

    def cut(flat):
        out, at = [], 3
        for n in sizes:
            out.append(flat[at:at + n])
            at += n
        return out

    p = torch.randn(total, generator=torch.Generator().manual_seed(1))
    fp, fg = p.to(DEV), torch.zeros(total, device=DEV)
    if bits == 32:
        fm, fv = torch.zeros(total, device=DEV), torch.zeros(total, device=DEV)
        artemis_amd.adamw_step(cut(fp), cut(fg), cut(fm), cut(fv), 5, **ARGS)
    else:
        fm, fv = (torch.zeros(total, dtype=torch.uint8, device=DEV) for _ in range(2))
        bases = [[torch.full(((n + 255) // 256,), 7, dtype=torch.int32, device=DEV) for n in sizes] for _ in range(2)]
        artemis_amd.adamw_step_8bit(cut(fp), cut(fg), cut(fm), bases[0], cut(fv), bases[1], 5, **ARGS)
    torch.cuda.synchronize()
    want = p * (1 - ARGS["lr"] * ARGS["weight_decay"])
    want[:3] = p[:3]
    assert torch.equal(fp.cpu(), want)
    assert not fm.any() and not fv.any()


def state8(m, v, seed):
    g = torch.Generator().manual_seed(seed)
    r = [torch.randint(0, 1 << 16, t.shape, generator=g) for t in m]
    return [[*ref.encode(a, z, True), *ref.encode(b, z, False)] for a, b, z in zip(m, v, r)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("step,seed", [(1, 0), (7, 103), (10 ** 6, 2 ** 32 - 1)])
def test_8_bits_bit_for_bit(dtype, step, seed):
    p, g, m, v = data(SIZES, dtype, step, spread=6)
    s = state8(m, v, 3)
    if step == 1:
        s = [[torch.zeros_like(t) for t in k] for k in s]
    dp, dg = on(p), on(g)
    ds = [on([k[i] for k in s]) for i in range(4)]
    artemis_amd.adamw_step_8bit(dp, dg, *ds, step, seed=seed, **ARGS)
    m2 = artemis_amd.moments_from_8bit(ds[0], ds[1], signed=True)
    v2 = artemis_amd.moments_from_8bit(ds[2], ds[3], signed=False)
    torch.cuda.synchronize()
    place = 0
    for i in range(len(p)):
        want = ref.adamw8(p[i], g[i], *s[i], step, place, seed, ARGS["lr"], ARGS["betas"], ARGS["eps"],
                          ARGS["weight_decay"])
        place += (p[i].numel() + 255) // 256
        for got, value, name in zip((dp[i], *(d[i] for d in ds)), want[:5], ("p", "m", "m base", "v", "v base")):
            assert torch.equal(got.cpu(), value), (name, i)
        assert torch.equal(m2[i].cpu(), ref.decode(want[1], want[2], True))
        assert torch.equal(v2[i].cpu(), ref.decode(want[3], want[4], False))


def test_codes_hold_what_they_say():
    """On the CPU: a code is within one step (an eighth of a binade) of the value, 0 stands for 0 alone in v, the largest value
    of a group fits, subnormals and huge values too; the mean over the random bits is the value."""
    g = torch.Generator().manual_seed(5)
    for scale in (1e-44, 1e-38, 1e-20, 1.0, 1e30, 3e38):
        v = torch.rand(1024, generator=g) * scale
        v[::7] *= 1e-4
        v[::11] = 0
        for r in (0, 1, 32768, 65535):
            random16 = torch.full(v.shape, r)
            for signed in (False, True):
                x = v * torch.where(torch.rand(v.shape, generator=g) < 0.5, -1.0, 1.0) if signed else v
                got = ref.decode(*ref.encode(x, random16, signed), signed)
                # a step at x: an eighth of its binade, or 2^-129 where the 11 bits run into the subnormals
                ax = x.abs().double()
                step = torch.maximum(torch.exp2(torch.floor(torch.log2(ax.clamp_min(2.0 ** -149)))) / 8,
                                     torch.tensor(2.0 ** -129, dtype=torch.float64))
                top = x.abs().view(-1, 256).amax(1).repeat_interleave(256)
                reach = 2.0 ** (-15 if signed else -30) * top.double()      # below: the smallest codes
                fine = ax >= torch.maximum(reach, torch.tensor(2.0 ** -125, dtype=torch.float64))
                assert ((got.double() - x.double()).abs()[fine] < step[fine] * (1 + 1e-12)).all()
                if not signed:
                    assert ((got > 0) == (x > 0)).all()
                assert (got.sign() * x.sign() >= 0).all()
    # every one of the 2^16 random values once: the mean of the decoded ones is the value, to 2^-16 of a step
    for x in (1.0, 0.7123, 0.333, 2.0 ** -14 * 1.3):
        group = torch.zeros(256)
        group[0], group[1] = 1.0, x
        for signed in (False, True):
            mean = 0.0
            base_code = [ref.encode(group, torch.full((256,), r), signed) for r in range(0, 65536, 257)]
            mean = sum(float(ref.decode(*c, signed)[1]) for c in base_code) / len(base_code)
            assert abs(mean - x) <= x / 8 / len(base_code) * 1.01 + x * 2.0 ** -16, (x, signed, mean)


def test_noise_is_even():
    """What the rounding at random needs of the generator.  A value a fraction f of a step above a code is rounded up where
    the half word u / 2^16 is at least 1 - f: with the probability 1 - F(1 - f), F the distribution function of
    the half words.  So the rounding's bias is at most a step times the largest distance of F from the even
    distribution's, whatever else the words' bits do (the low 8 bits of a half by themselves come out uneven at 2^20
    counters, chi square 391 for 255 degrees of freedom: that moves F within one 256th of the range, and the distance
    counts it).  For n even random words that distance is over 2.5 / sqrt(n) with probability 2 exp(-2 * 2.5^2) = 7e-6.
    A step of v is at most v / 8, so that at n = 2^20 the bias stays under v * 2.5 / 1024 / 8 = v * 3e-4 for one
    step's words, of another sign the next step.  Neighbours and halves: uncorrelated to six deviations."""
    n = 1 << 20
    even = (torch.arange(65536) + 1).double() / 65536
    for step, seed in ((1, 0), (2, 0), (1000, 103)):
        z = ref.noise(n, 0, step, seed)
        for half in (z & 0xFFFF, z >> 16):
            distance = float((torch.bincount(half, minlength=65536).cumsum(0).double() / n - even).abs().max())
            assert distance < 2.5 / 1024, (step, seed, distance)
            u = half.double() / 65536 - 0.5
            corr = float((u[1:] * u[:-1]).mean() * 12)
            assert abs(corr) < 6 / 1024, corr
        a, b = (z & 0xFFFF).double() / 65536 - 0.5, (z >> 16).double() / 65536 - 0.5
        assert abs(float((a * b).mean() * 12)) < 6 / 1024


@pytest.mark.gpu
def test_a_slow_second_moment_moves():
    """b2 = 0.999 from v = 1 towards g^2 = 4: after 1000 steps v = 4 - 3 * 0.999^1000 = 2.897.  Rounded to the nearest of 8
    steps in a binade it would stay 1.  Each step rounds by less than a step s <= v / 8, at random without bias,
    and decays by 0.999 a step after: the standard deviation of an element is at most sqrt(sum 0.999^(2k)) * s / 2
    <= 22.4 * 0.5 / 2; the mean over 65536 elements is off by at most 6 / 256 of that."""
    n = 65536
    p, g = [torch.zeros(n, device=DEV)], [torch.full((n,), 2.0, device=DEV)]
    ones = torch.ones(n)
    mc, mb = ref.encode(torch.zeros(n), torch.zeros(n, dtype=torch.long), True)
    vc, vb = ref.encode(ones, torch.zeros(n, dtype=torch.long), False)
    s = [[t.to(DEV)] for t in (mc, mb, vc, vb)]
    for t in range(1, 1001):
        artemis_amd.adamw_step_8bit(p, g, *s, t, lr=0.0, seed=1)
    v, = artemis_amd.moments_from_8bit(s[2], s[3], signed=False)
    mean = float(v.double().mean())
    assert abs(mean - (4 - 3 * 0.999 ** 1000)) < 22.4 * 0.5 / 2 * 6 / 256, mean


@pytest.mark.gpu
def test_gradients_that_are_not_finite():
    p, g, m, v = data([600], torch.float32, 3)
    g[0][300] = float("inf")
    s = state8(m, v, 1)
    dp, dg, ds = on(p), on(g), [on([k[i] for k in s]) for i in range(4)]
    artemis_amd.adamw_step_8bit(dp, dg, *ds, 3, **ARGS)
    v2, = artemis_amd.moments_from_8bit(ds[2], ds[3], signed=False)
    assert v2[0, ].isfinite() and v2[300].isinf() and dp[0][300].isnan()
    assert v2[:256].isfinite().all() and v2[512:].isfinite().all()           # the other groups
    assert dp[0].isnan().sum() == 1
    g[0][300] = float("nan")
    dp, dg, dm, dv = on(p), on(g), on(m), on(v)
    artemis_amd.adamw_step(dp, dg, dm, dv, 3, **ARGS)
    assert dp[0].isnan().sum() == 1 and dm[0].isnan().sum() == 1 and dv[0].isnan().sum() == 1


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer(bits):
    """Two groups, parameters without a gradient, mixed types; against the function, and saved and loaded half-way."""
    g = torch.Generator().manual_seed(1)

    def make():
        r = torch.Generator().manual_seed(2)
        return [torch.nn.Parameter(torch.randn(s, generator=r).to(t).to(DEV)) for s, t in
                [((3, 5), torch.float32), ((700,), torch.float32), ((2, 4097), torch.bfloat16), ((9,), torch.float32)]]

    def groups(ps):
        return [{"params": ps[:2]}, {"params": ps[2:], "lr": 1e-2, "weight_decay": 0.0}]

    ps = make()
    opt = AdamW(groups(ps), lr=1e-3, moment_bits=bits, seed=9)
    again, opt2 = make(), None
    for t in range(6):
        grads = [torch.randn(p.shape, generator=g).to(p.dtype).to(DEV) for p in ps]
        if t == 3:
            opt2 = AdamW(groups(again), lr=5.0, moment_bits=bits)
            opt2.load_state_dict(torch.load(_saved(opt.state_dict()), weights_only=True))
            for a, b in zip(again, ps):
                a.data.copy_(b.data)
        for o, qs in ((opt, ps), (opt2, again)):
            if o is None:
                continue
            for i, (q, gr) in enumerate(zip(qs, grads)):
                q.grad = None if i == 3 or (i == 1 and t == 0) else gr.clone()
            o.step()
    for a, b in zip(ps, again):
        assert torch.equal(a, b)
        for name, value in opt.state[a].items():
            other = opt2.state[b][name]
            assert value == other if name == "step" else (torch.equal(value, other) and value.dtype == other.dtype)
    assert opt.state[ps[0]]["step"] == 6 and opt.state[ps[1]]["step"] == 5 and not opt.state[ps[3]]
    assert torch.equal(ps[3], make()[3])


def _saved(state):
    import io
    f = io.BytesIO()
    torch.save(state, f)
    f.seek(0)
    return f


@pytest.mark.gpu
def test_follows_the_stock_optimizer():
    """fp32, 20 steps: both round a handful of times in a step, and the update is at most lr / (1 - b1) long, so that after
    20 steps they differ by 20 * 16 u (|p| + 10 lr) at most; a sign where a moment is all rounding is damped by eps."""
    r = torch.Generator().manual_seed(4)
    a = [torch.nn.Parameter(torch.randn(s, generator=r).to(DEV)) for s in (100, 5000)]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    ours = AdamW(a, lr=1e-3, weight_decay=0.1, eps=1e-3)
    stock = torch.optim.AdamW(b, lr=1e-3, weight_decay=0.1, eps=1e-3, foreach=False, fused=False)
    for _ in range(20):
        for p, q in zip(a, b):
            p.grad = torch.randn(p.shape, generator=r).to(DEV)
            q.grad = p.grad.clone()
        ours.step(), stock.step()
    for p, q in zip(a, b):
        ref.assert_within(p, q, 20 * 16 * ref.U * (q.abs() + 1e-2), "p")


@pytest.mark.gpu
def test_a_step_is_not_captured():
    p, g, m, v = (on(t) for t in data([100], torch.float32, 3))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError, match="captured"):
            artemis_amd.adamw_step(p, g, m, v, 1)
        p[0].mul_(1.0)


def test_refusals():
    def lists(n=2, dtype=torch.float32):
        return [[torch.zeros(300, dtype=dtype) for _ in range(n)] for _ in range(4)]

    p, g, m, v = lists()
    with pytest.raises(NotImplementedError):
        artemis_amd.adamw_step(p, g, m, v, 1)
    artemis_amd.adamw_step([], [], [], [], 1)
    assert artemis_amd.moments_from_8bit([], [], True) == []
    with pytest.raises(ValueError):
        artemis_amd.adamw_step(p, g[:1], m, v, 1)
    with pytest.raises(ValueError):
        artemis_amd.adamw_step(p, [g[0], g[1][:299]], m, v, 1)
    for step, error in ((0, ValueError), (-1, ValueError), (1.5, TypeError)):
        with pytest.raises(error):
            artemis_amd.adamw_step(p, g, m, v, step)
    with pytest.raises(ValueError, match="twice"):
        artemis_amd.adamw_step([p[0], p[0]], g, m, v, 1)
    with pytest.raises(ValueError, match="twice"):
        artemis_amd.adamw_step(p, g, [m[0], m[0]], v, 1)
    with pytest.raises(TypeError):
        artemis_amd.adamw_step(*lists(dtype=torch.float64), 1)
    with pytest.raises(TypeError):
        artemis_amd.adamw_step(p, [t.half() for t in g], m, v, 1)
    with pytest.raises(TypeError):
        artemis_amd.adamw_step(p, g, [t.half() for t in m], v, 1)
    with pytest.raises(AssertionError):
        artemis_amd.adamw_step([torch.zeros(20, 15).t(), p[1]], g, m, v, 1)
    codes, bases = [torch.zeros(300, dtype=torch.uint8)], [torch.zeros(2, dtype=torch.int32)]
    with pytest.raises(NotImplementedError):
        artemis_amd.adamw_step_8bit(p[:1], g[:1], codes, bases, [codes[0].clone()], [bases[0].clone()], 1)
    with pytest.raises(ValueError):
        artemis_amd.adamw_step_8bit(p[:1], g[:1], codes, [bases[0][:1]], [codes[0].clone()], bases, 1)
    with pytest.raises(TypeError):
        artemis_amd.moments_from_8bit([codes[0].int()], bases, True)
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-1.0),
               dict(moment_bits=16), dict(lr=math.nan)):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(torch.zeros(3))], **kw)


def test_a_tensor_for_two_purposes_is_refused():
    p, g, m, v = ([torch.zeros(300)] for _ in range(4))
    for lists in ((p, g, p, v), (p, g, m, m), (p, g, m, p)):
        with pytest.raises(ValueError, match="twice"):
            artemis_amd.adamw_step(*lists, 1)
    c, d = ([torch.zeros(300, dtype=torch.uint8)] for _ in range(2))
    bases = [torch.zeros(2, dtype=torch.int32)]
    with pytest.raises(ValueError, match="twice"):
        artemis_amd.adamw_step_8bit(p, g, c, bases, d, bases, 1)


def test_a_refused_step_is_not_counted_and_groups_are_checked():
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    optimizer = AdamW([p])
    with pytest.raises(NotImplementedError):
        optimizer.step()                                         # (a parameter on the CPU)
    assert optimizer.state[p]["step"] == 0
    for kw in (dict(moment_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9))):
        with pytest.raises(ValueError):
            optimizer.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2))], **kw})
    assert len(optimizer.param_groups) == 1
