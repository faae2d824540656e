"""Group norm, rotary positions and cross attention on device arrays, against their formulas in 64 bits.

Tolerances follow from the arithmetic.  U[t] is half a step of type t relative to the value (one rounding to it).
F = 2^-24 is fp32's; a sum of n terms in fp32 is off by at most n F times the sum of their magnitudes in any order.
"""
import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}  # half the smallest step: subnormal results round by this much
F = 2.0 ** -24
KIND = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPES = ["f32", "f16", "bf16"]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def assert_within(got, want, bound):
    got = got.double()
    bad = int((~torch.isfinite(got)).sum())
    assert bad == 0, bad
    over = (got - want).abs() - bound
    worst = int(over.argmax())
    assert over.max() <= 0, (float(got.flatten()[worst]), float(want.flatten()[worst]), float(bound.expand_as(want).flatten()[worst]))


# ------------------------------------------------------------------------------------------------ refusals (no GPU)
def status_of(call):
    with pytest.raises(Exception) as err:
        call()
    return getattr(err.value, "status", type(err.value).__name__)


def host(n=64):
    a = np.zeros(n, np.float32)
    return a, a.ctypes.data


def test_arrays_that_start_between_elements_are_refused(pkg):
    keep = [host() for _ in range(4)]
    a, b, c, d = (x[1] for x in keep)
    for at in range(4):
        p = [a, b, c, d]
        p[at] += 1 if at < 2 else 2
        assert status_of(lambda: pkg.op_group_norm(p[0], p[1], "bf16", 1, 2, 4, 2, p[2], p[3])) == 2
        with pytest.raises(pkg.NcnnB200Error, match="start"):
            pkg.op_cross_attention(*[x + (1 if n == at else 0) for n, x in enumerate((a, b, c, d))], "f16", 1, 1, 1, 1, 1, 8)
    with pytest.raises(pkg.NcnnB200Error, match="start"):
        pkg.op_cross_attention(a, b, c, d, "f16", 1, 1, 1, 1, 1, 8, kv_lens_ptr=a + 2)
    for x, y, p in ((a + 2, b, c), (a, b + 2, c), (a, b, c + 2)):
        with pytest.raises(pkg.NcnnB200Error, match="start"):
            pkg.op_rotary_axes(x, y, "f32", 1, 1, 8, p, [2])


def test_group_norm_refuses(pkg):
    a, p = host()
    b, r = host()
    ok = dict(element="f32", n=1, pixels=4, channels=8, groups=2)

    def call(x=p, y=r, gamma=None, beta=None, eps=1e-5, act="none", xp=0, yp=0, **kw):
        v = {**ok, **kw}
        return lambda: pkg.op_group_norm(x, y, v["element"], v["n"], v["pixels"], v["channels"], v["groups"], gamma, beta, eps, act, xp, yp)

    assert status_of(call(x=None)) == 1 and status_of(call(y=None)) == 1
    for bad in (dict(n=-1), dict(pixels=-1), dict(channels=0), dict(groups=0), dict(groups=3), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf),
                dict(xp=7), dict(yp=7), dict(x=p, y=p, xp=9, yp=10)):
        assert status_of(call(**bad)) == 2, bad
    assert status_of(call(pixels=1 << 40)) == 4
    assert status_of(call(element="f64")) == "ValueError" and status_of(call(act="cube")) == "ValueError"
    # an array that kernels cannot reach is refused, not read
    with pytest.raises(pkg.NcnnB200Error) as err:
        call()()
    assert err.value.status == 2 and "device memory" in str(err.value)
    call(n=0)()
    call(pixels=0)()


def test_rotary_refuses(pkg):
    a, p = host()
    b, r = host()

    def call(x=p, y=r, element="f32", tokens=2, heads=1, d=8, positions=p, sections=(2, 2), base=10000.0, strides=None):
        return lambda: pkg.op_rotary_axes(x, y, element, tokens, heads, d, positions, sections, base, strides=strides)

    assert status_of(call(x=None)) == 1 and status_of(call(y=None)) == 1 and status_of(call(positions=None)) == 1
    for bad in (dict(tokens=-1), dict(heads=0), dict(d=0), dict(sections=()), dict(sections=(0, 0)), dict(sections=(3, -1)), dict(sections=(3, 2)),
                dict(sections=(1, 1, 1, 1, 0)), dict(sections=(64, 65), d=512), dict(base=0.5), dict(base=math.nan), dict(base=math.inf),
                dict(strides=(8, 8, 7, 8)), dict(strides=(-8, 8, 8, 8)), dict(heads=2, strides=(16, 8, 16, 4)), dict(x=p, y=p, strides=(16, 8, 8, 8))):
        assert status_of(call(**bad)) == 2, bad
    assert status_of(call(tokens=1 << 31, heads=1 << 10)) == 4
    for at in range(4):
        assert status_of(call(strides=[1 << 62 if n == at else 8 for n in range(4)])) == 4
    assert status_of(call(strides=(1, 2, 3))) == "ValueError"
    with pytest.raises(pkg.NcnnB200Error) as err:
        call()()
    assert err.value.status == 2 and "device memory" in str(err.value)
    call(tokens=0)()


def test_cross_attention_refuses(pkg):
    keep = [host() for _ in range(4)]
    q, k, v, o = (x[1] for x in keep)

    def call(q=q, k=k, v=v, o=o, element="f32", b=1, lq=2, lk=3, heads=2, kv_heads=1, d=8, scale=0.0, strides=None):
        return lambda: pkg.op_cross_attention(q, k, v, o, element, b, lq, lk, heads, kv_heads, d, None, None, scale, strides)

    assert [status_of(call(**{n: None})) for n in "qkvo"] == [1] * 4
    dense = (32, 16, 8, 24, 8, 8, 24, 8, 8, 32, 16, 8)
    for bad in (dict(b=-1), dict(lq=-1), dict(lk=-1), dict(heads=0), dict(kv_heads=0), dict(heads=3, kv_heads=2), dict(d=0), dict(d=257), dict(b=65536),
                dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(o=q), dict(o=k), dict(o=v),
                dict(strides=dense[:9] + (32, 16, 7)), dict(strides=dense[:9] + (0, 8, 4)), dict(strides=(-32,) + dense[1:])):
        assert status_of(call(**bad)) == 2, bad
    assert status_of(call(strides=(1 << 60,) + dense[1:])) == 4
    assert status_of(call(strides=dense[:4])) == "ValueError"
    with pytest.raises(pkg.NcnnB200Error) as err:
        call()()
    assert err.value.status == 2 and "device memory" in str(err.value)
    call(b=0)()
    call(lq=0)()


# ------------------------------------------------------------------------------------------------ group norm
ACTS = {"none": lambda a: a, "relu": torch.relu, "swish": lambda a: a * torch.sigmoid(a), "gelu": lambda a: a * torch.special.ndtr(a)}


def norm_want(x, groups, gamma, beta, eps, act):
    """The result, and how far fp32 statistics and one rounding to the type may take it."""
    n, p, c = x.shape
    t = x.double().view(n, p, groups, c // groups)
    mean = t.mean((1, 3), keepdim=True)
    var = (t - mean).square().mean((1, 3), keepdim=True)
    z = (t - mean) / torch.sqrt(var + eps)
    g = torch.ones(c, device="cuda", dtype=torch.float64) if gamma is None else gamma.double()
    b = torch.zeros(c, device="cuda", dtype=torch.float64) if beta is None else beta.double()
    # mean: threads sum at most 2^9 terms each and a tree of 2^5 joins them, so it is off by 2^10 F of the mean magnitude
    # at most; the variance by as much of itself, relatively, and by the mean's error squared
    dm = 2.0 ** 10 * F * t.abs().mean((1, 3), keepdim=True) / torch.sqrt(var + eps)
    off = ((dm + z.abs() * (2.0 ** 10 * F + dm * dm) + 4 * F * (z.abs() + mean.abs() / torch.sqrt(var + eps))).view(n, p, c)) * g.abs()
    pre = z.view(n, p, c) * g + b
    # an activation here is at most 1.13 times as steep as the line; exp and erfc are good to a few F of their argument's size
    return ACTS[act](pre), 1.13 * (off + 2 * F * (pre.abs() + b.abs())) + 16 * F * (1 + pre.abs()) * pre.abs()


def check_norm(pkg, element, n, p, c, groups, act, affine=True, offset=1.0, eps=1e-5, x_pitch=0, y_pitch=0, in_place=False, shift=0, seed=0):
    g = gen(seed)
    xp, yp = x_pitch or c, y_pitch or c
    wide = (normal(g, n * p * xp + shift) * 1.5 + offset).to(KIND[element])
    out = torch.full((n * p * yp + shift,), 7.0, device="cuda", dtype=KIND[element])
    x = wide[shift:].view(n, p, xp)[:, :, :c].clone()
    gamma, beta = (normal(g, c), normal(g, c)) if affine else (None, None)
    size = wide.element_size()
    to = wide if in_place else out
    before = to.clone()
    pkg.op_group_norm(wide.data_ptr() + shift * size, to.data_ptr() + shift * size, element, n, p, c, groups,
                      None if gamma is None else gamma.data_ptr(), None if beta is None else beta.data_ptr(), eps, act, x_pitch, y_pitch)
    torch.cuda.synchronize()
    want, off = norm_want(x, groups, gamma, beta, eps, act)
    got = to[shift:].view(n, p, yp)
    assert_within(got[:, :, :c], want, off + U[element] * (want.abs() + off) + TINY[element])
    # what lies between the rows and in front of them stays
    assert torch.equal(got[:, :, c:], before[shift:].view(n, p, yp)[:, :, c:]) and torch.equal(to[:shift], before[:shift])


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("n,p,c,groups,act", [(1, 1, 1, 1, "none"), (1, 1, 8, 2, "none"), (2, 49, 512, 32, "swish"), (3, 33 * 47, 91, 7, "gelu"),
                                              (2, 1000, 320, 32, "swish"), (1, 5000, 40, 1, "relu"), (1, 300, 64, 64, "none"), (5, 17, 24, 3, "relu"),
                                              (1, 20000, 128, 32, "swish"), (2, 4096, 8, 1, "none"), (1, 100, 2560, 32, "swish"), (16, 1, 96, 4, "gelu"),
                                              (1, 70000, 12, 4, "none"), (2, 640, 1030, 10, "swish"), (1, 9, 5000, 5, "none")])
def test_group_norm(pkg, element, n, p, c, groups, act):
    check_norm(pkg, element, n, p, c, groups, act)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
def test_group_norm_layouts(pkg, element):
    """No affine, ranges of wider tensors' channels, addresses of one element's alignment, in place."""
    check_norm(pkg, element, 2, 200, 64, 8, "relu", affine=False)
    check_norm(pkg, element, 2, 200, 64, 8, "swish", x_pitch=96, y_pitch=72)
    check_norm(pkg, element, 2, 200, 64, 8, "swish", x_pitch=97, y_pitch=64, shift=1)
    check_norm(pkg, element, 2, 300, 33, 3, "none", x_pitch=40, y_pitch=41, shift=3)
    check_norm(pkg, element, 3, 2000, 160, 32, "swish", in_place=True)
    check_norm(pkg, element, 1, 30000, 64, 32, "none", in_place=True, x_pitch=80, y_pitch=80)


@pytest.mark.gpu
def test_group_norm_far_from_zero(pkg):
    """A mean of a thousand deviations: sums of squares about zero would lose the variance."""
    g = gen(3)
    x = (normal(g, 2, 3000, 32) + 1000.0)
    y = torch.empty_like(x)
    pkg.op_group_norm(x.data_ptr(), y.data_ptr(), "f32", 2, 3000, 32, 4, None, None, 1e-5, "none")
    t = x.double().view(2, 3000, 4, 8)
    d, m = torch.std_mean(t, (1, 3), keepdim=True, correction=0)
    want = ((t - m) / torch.sqrt(d * d + 1e-5)).view(2, 3000, 32)
    # the mean's error (2^10 F of 1000 at most, see norm_want) moves every value; the variance takes its square
    assert_within(y, want, 2.0 ** 10 * F * 1000 + want.abs() * (2.0 ** 10 * F * 2 + (2.0 ** 10 * F * 1000) ** 2) + 4 * F * 1000)


@pytest.mark.gpu
def test_group_norm_constant_and_nonfinite(pkg):
    """A group of one value is beta (variance 0); a NaN or an infinity stays in its own group of its own image."""
    x = torch.full((2, 700, 16), 3.0, device="cuda")
    x[1] = normal(gen(1), 700, 16)
    x[1, 5, 2] = math.nan
    x[1, 9, 14] = math.inf
    y = torch.empty_like(x)
    beta = torch.arange(16, device="cuda", dtype=torch.float32)
    pkg.op_group_norm(x.data_ptr(), y.data_ptr(), "f32", 2, 700, 16, 4, None, beta.data_ptr(), 1e-5, "relu")
    assert torch.equal(y[0], beta.expand(700, 16))
    assert torch.isnan(y[1, :, 0:4]).all() and torch.isnan(y[1, 9, 14]) and torch.isfinite(y[1, :, 4:12]).all()


@pytest.mark.gpu
def test_group_norm_is_the_same_every_time(pkg):
    x = normal(gen(8), 4, 5000, 96)
    ys = []
    for _ in range(3):
        y = torch.empty_like(x)
        pkg.op_group_norm(x.data_ptr(), y.data_ptr(), "f32", 4, 5000, 96, 12, None, None, 1e-5, "swish")
        ys.append(y)
    assert torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[2])
    one = torch.empty_like(x[2])
    pkg.op_group_norm(x[2].data_ptr(), one.data_ptr(), "f32", 1, 5000, 96, 12, None, None, 1e-5, "swish")
    # an image alone is summed over other ranges of pixels: the same value, not the same bits
    assert (one - ys[0][2]).abs().max() <= 2.0 ** 12 * F


# ------------------------------------------------------------------------------------------------ rotary positions
def rotary_want(x, positions, sections, base, interleaved, shared):
    y = x.double().clone()
    size = torch.zeros_like(y)
    pairs, first = sum(sections), 0
    for a, count in enumerate(sections):
        for j in range(count):
            rate = float(base) ** -((first + j) / pairs if shared else j / count)
            turn = torch.remainder(positions[:, a].double() * rate, 2 * math.pi)
            c, s = torch.cos(turn)[:, None], torch.sin(turn)[:, None]
            i = first + j
            at = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
            u, v = x[..., at[0]].double(), x[..., at[1]].double()
            y[..., at[0]], y[..., at[1]] = u * c - v * s, u * s + v * c
            size[..., at[0]] = size[..., at[1]] = u.abs() + v.abs()
        first += count
    return y, size


def check_rotary(pkg, element, tokens, heads, d, sections, interleaved, shared, far=1000, base=10000.0, rows=0, strides=None, in_place=False, shift=0,
                 low=None):
    g = gen(tokens + heads)
    xs = (heads * d, d, heads * d, d) if strides is None else strides
    buffers = []
    for t, h in (xs[:2], xs[2:]):
        buffers.append(normal(g, (tokens - 1) * t + (heads - 1) * h + d + shift).to(KIND[element]))
    src, dst = buffers
    if in_place:
        dst = src
    x = torch.as_strided(src, (tokens, heads, d), (xs[0], xs[1], 1), shift).clone()
    before = dst.clone()
    r = rows or tokens
    positions = torch.randint(-far if low is None else low, far, (r, len(sections)), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    size = src.element_size()
    pkg.op_rotary_axes(src.data_ptr() + shift * size, dst.data_ptr() + shift * size, element, tokens, heads, d, positions.data_ptr(), sections, base,
                       interleaved, shared, rows, strides)
    torch.cuda.synchronize()
    at = positions[torch.arange(tokens, device="cuda") % r]
    want, mag = rotary_want(x, at, sections, base, interleaved, shared)
    got = torch.as_strided(dst, (tokens, heads, d), (xs[2], xs[3], 1), shift)
    # the angle's fp32 half turns are off by F of themselves (pi F at most), sine and cosine by 2 F more, the products by F each;
    # the reference's own angle in double by 2^-52 of it
    assert_within(got, want, (math.pi + 6) * F * mag + far * 2.0 ** -51 * mag + U[element] * (want.abs() + 10 * F * mag) + TINY[element])
    left = torch.ones_like(dst, dtype=torch.bool)
    torch.as_strided(left, (tokens, heads, d), (xs[2], xs[3], 1), shift).fill_(False)
    assert torch.equal(dst[left], before[left])
    assert torch.equal(got[..., 2 * sum(sections):], x[..., 2 * sum(sections):])


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,d,sections,shared", [(1, 1, 2, [1], False), (1, 32, 128, [16, 24, 24], True), (77, 5, 72, [16, 16], False),
                                                            (33, 3, 26, [9, 4], True), (4097, 24, 128, [22, 21, 21], False), (500, 7, 40, [5, 5, 5, 5], True),
                                                            (3, 2, 256, [128], False), (1000, 16, 80, [0, 20, 20], False), (19, 4, 18, [9], True)])
def test_rotary(pkg, element, interleaved, tokens, heads, d, sections, shared):
    check_rotary(pkg, element, tokens, heads, d, sections, interleaved, shared)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_layouts(pkg, element, interleaved):
    """The heads of a joint projection, head-major results, one element's alignment, in place, positions that repeat."""
    check_rotary(pkg, element, 300, 8, 64, [16, 16], interleaved, False, strides=(24 * 64, 64, 8 * 64, 64))
    check_rotary(pkg, element, 300, 8, 64, [16, 16], interleaved, False, strides=(8 * 64, 64, 64, 300 * 64))
    check_rotary(pkg, element, 50, 3, 24, [6, 6], interleaved, True, strides=(75, 25, 73, 24), shift=1)
    check_rotary(pkg, element, 1200, 12, 64, [8, 12, 12], interleaved, False, in_place=True)
    check_rotary(pkg, element, 1200, 12, 64, [8, 8], interleaved, False, in_place=True, strides=(36 * 64, 64, 36 * 64, 64))
    check_rotary(pkg, element, 600, 4, 32, [8, 8], interleaved, False, rows=150)


@pytest.mark.gpu
def test_rotary_far_positions(pkg):
    """Positions up to the ends of their type keep their angles (fp32 products would lose them altogether)."""
    check_rotary(pkg, "f32", 2000, 4, 64, [32], True, False, far=(1 << 31) - 1, low=-(1 << 31))
    check_rotary(pkg, "f32", 2000, 4, 64, [16, 16], False, True, far=1000000, base=500000.0)
    check_rotary(pkg, "f32", 64, 4, 64, [16, 16], False, True, far=100, base=1.0)


# ------------------------------------------------------------------------------------------------ cross attention
def attend_want(q, k, v, keep, scale, element):
    """The result and its tolerance.  keep: [batch][lk] booleans."""
    b, lq, heads, d = q.shape
    shared = heads // k.shape[2]
    o = torch.zeros(b, lq, heads, d, device="cuda", dtype=torch.float64)
    bound = torch.zeros_like(o)
    for i in range(b):
        at = keep[i].nonzero().flatten()
        if at.numel() == 0:
            continue
        for h in range(heads):
            qq, kk, vv = q[i, :, h].double(), k[i, at, h // shared].double(), v[i, at, h // shared].double()
            s = qq @ kk.T * scale
            p = torch.softmax(s, -1)
            o[i, :, h] = p @ vv
            spread = p @ vv.abs()
            # a score: d products summed in fp32 (truncated sums may lose 2 F a term), its scaling and its difference to the
            # maximum 8 F of the sizes; a probability is off by as much, the sum over the keys by 2 lk F; 16-bit types round
            # each probability once (U of it); then the result's own rounding
            ds = (2 * d + 8) * F * ((qq.abs() @ kk.abs().T) * scale).amax(-1, keepdim=True) + 8 * F * s.abs().amax(-1, keepdim=True)
            rel = 2 * ds + 4 * at.numel() * F + 16 * F + (U[element] if element != "f32" else 0.0)
            # probabilities under the type's smallest step (fp16) vanish: 2^-25 of the largest a key
            lost = 2.0 ** -25 * at.numel() * vv.abs().amax() if element == "f16" else 0.0
            bound[i, :, h] = rel * spread + lost + U[element] * (o[i, :, h].abs() + rel * spread) + TINY[element]
    return o, bound


def check_attend(pkg, element, b, lq, lk, heads, kv_heads, d, lens=None, mask=None, scale=0.0, seed=0, spread=1.5, junk=True, strides=None, shift=0):
    g = gen(seed + lq + lk)
    if strides is None:
        strides = (lq * heads * d, heads * d, d, lk * kv_heads * d, kv_heads * d, d, lk * kv_heads * d, kv_heads * d, d, lq * heads * d, heads * d, d)
        packed = None
    else:
        packed = strides
    shapes = [(b, lq, heads, d), (b, lk, kv_heads, d), (b, lk, kv_heads, d), (b, lq, heads, d)]
    buffers, views = [], []
    for n, shape in enumerate(shapes):
        st = strides[3 * n:3 * n + 3]
        size = sum((e - 1) * s for e, s in zip(shape, st)) + d + shift if 0 not in shape else shift
        buf = normal(g, size).to(KIND[element])
        buffers.append(buf)
        views.append(torch.as_strided(buf, shape, (*st, 1), shift) if 0 not in shape else buf.new_empty(shape))
    q, k, v, o = views
    q.mul_(spread)
    keep = torch.ones(b, lk, dtype=torch.bool, device="cuda")
    lens_t = mask_t = None
    if lens is not None:
        lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
        keep &= torch.arange(lk, device="cuda")[None] < lens_t[:, None]
    if mask is not None:
        mask_t = mask.to("cuda").to(torch.uint8).contiguous()
        keep &= mask_t.bool()
    if junk and (lens is not None or mask is not None) and all(s > 0 for s in strides):
        # what lies at keys without a part is never used
        k[~keep] = math.nan
        v[~keep] = math.inf
        v[~keep, :, ::2] = math.nan
    before = buffers[3].clone()
    size = buffers[0].element_size()
    pkg.op_cross_attention(*[t.data_ptr() + shift * size for t in buffers], element, b, lq, lk, heads, kv_heads, d,
                           None if lens_t is None else lens_t.data_ptr(), None if mask_t is None else mask_t.data_ptr(), scale, packed)
    torch.cuda.synchronize()
    want, bound = attend_want(q, k, v, keep, scale or 1 / math.sqrt(d), element)
    assert_within(o, want, bound)
    left = torch.ones_like(buffers[3], dtype=torch.bool)
    torch.as_strided(left, shapes[3], (*strides[9:], 1), shift).fill_(False)
    assert torch.equal(buffers[3][left], before[left])
    return o


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("b,lq,lk,heads,kv_heads,d", [
    (1, 1, 1, 1, 1, 8), (1, 1, 1500, 16, 16, 64), (3, 1, 700, 32, 8, 128), (2, 2, 129, 8, 1, 64), (1, 5, 64, 6, 2, 40), (2, 17, 77, 4, 4, 80),
    (1, 128, 128, 2, 2, 64), (1, 129, 127, 2, 1, 128), (2, 300, 77, 5, 5, 64), (1, 1000, 333, 8, 8, 40), (1, 257, 640, 3, 3, 96), (1, 64, 1, 2, 2, 128),
    (1, 200, 300, 2, 2, 160), (1, 130, 260, 2, 1, 256), (1, 3, 1000, 2, 1, 192), (1, 7, 50, 3, 3, 1), (2, 33, 45, 2, 2, 13), (1, 600, 513, 4, 2, 32),
    (1, 1, 20000, 2, 1, 128), (4, 1, 33, 64, 2, 72), (1, 16, 4096, 8, 8, 64), (1, 40, 3000, 4, 1, 128), (1, 1, 5, 128, 1, 64)])
def test_cross_attention(pkg, element, b, lq, lk, heads, kv_heads, d):
    check_attend(pkg, element, b, lq, lk, heads, kv_heads, d)


LENGTHS = [(1, 4, 1000), (200, 4, 500), (300, 4, 129), (1, 4, 64), (20, 4, 257)]


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("d", [40, 64, 128, 160])
@pytest.mark.parametrize("lq,b,lk", LENGTHS)
def test_cross_attention_lengths(pkg, element, d, lq, b, lk):
    """Ragged sequences, none of them and more than all of them, NaN and infinities behind their ends."""
    o = check_attend(pkg, element, b, lq, lk, 4, 2, d, lens=[0, 1, lk // 2 + 1, lk + 5])
    assert not o[0].any()
    check_attend(pkg, element, b, lq, lk, 4, 4, d, lens=[-3, 63, 65, lk - 1])


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("d", [40, 64, 128, 160])
@pytest.mark.parametrize("lq,b,lk", LENGTHS)
def test_cross_attention_masks(pkg, element, d, lq, b, lk):
    """Masks with holes, without any key, with one key, over a whole tile; alone and with lengths."""
    mask = torch.rand(b, lk, generator=torch.Generator().manual_seed(lk)) < 0.5
    mask[1] = False
    mask[2] = False
    mask[2, lk - 1] = True
    mask[3, : min(lk - 1, 128)] = False
    o = check_attend(pkg, element, b, lq, lk, 4, 2, d, mask=mask)
    assert not o[1].any()
    mask[0, lk // 2:] = False
    check_attend(pkg, element, b, lq, lk, 2, 2, d, mask=mask, lens=[lk, lk, lk - 1, lk // 2 + 1])


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("d,lk", [(64, 77), (40, 128), (128, 100), (72, 33), (64, 16), (128, 1)])
def test_cross_attention_text(pkg, element, d, lk):
    """Many queries over few keys, more tiles than SMs: whole sequences, ragged ones, one without keys, masks with holes."""
    check_attend(pkg, element, 4, 700, lk, 8, 4, d)
    check_attend(pkg, element, 5, 650, lk, 8, 8, d, lens=[lk, 0, 1, lk // 2 + 1, 0])
    mask = torch.rand(5, lk, generator=torch.Generator().manual_seed(lk)) < 0.5
    mask[3] = False
    check_attend(pkg, element, 5, 650, lk, 8, 2, d, mask=mask, lens=[lk, lk, lk // 2 + 1, lk, lk - 1])


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("lq", [1, 150])
def test_cross_attention_layouts(pkg, element, lq):
    """Head-major arrays, slices of a joint projection, keys that all heads or all sequences share, one element's alignment."""
    b, lk, h, d = 2, 200, 4, 64
    major = (h * lq * d, d, lq * d, h * lk * d, d, lk * d, h * lk * d, d, lk * d, h * lq * d, d, lq * d)
    check_attend(pkg, element, b, lq, lk, h, h, d, strides=major)
    joint = (lq * 3 * h * d, 3 * h * d, d, lk * 3 * h * d, 3 * h * d, d, lk * 3 * h * d, 3 * h * d, d, lq * h * d, h * d, d)
    check_attend(pkg, element, b, lq, lk, h, h, d, strides=joint)
    same = (lq * h * d, h * d, d, 0, d, 0, 0, d, 0, lq * h * d, h * d, d)
    check_attend(pkg, element, b, lq, lk, h, h, d, strides=same)
    odd = (lq * (h * d + 3), h * d + 3, d, lk * (h * d + 1), h * d + 1, d, lk * h * d, h * d, d, lq * h * d + 5, h * d, d)
    check_attend(pkg, element, b, lq, lk, h, h, d, strides=odd, shift=1, lens=[77, 200], junk=False)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
def test_cross_attention_scores(pkg, element):
    """Sharp and flat distributions, scales of one's own, maxima that rise along the keys."""
    check_attend(pkg, element, 1, 70, 400, 2, 2, 64, spread=20.0)
    check_attend(pkg, element, 1, 70, 400, 2, 2, 64, spread=0.01)
    check_attend(pkg, element, 1, 70, 400, 2, 2, 64, scale=1.0, spread=1.0)
    for lq in (1, 140):
        b, lk, d = 1, 900, 64
        q = torch.ones(b, lq, 2, d, device="cuda", dtype=KIND[element])
        k = (torch.arange(lk, device="cuda").view(1, lk, 1, 1) * 0.01).expand(b, lk, 2, d).to(KIND[element]).contiguous()
        v = normal(gen(1), b, lk, 2, d).to(KIND[element])
        o = torch.empty_like(q)
        pkg.op_cross_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), element, b, lq, lk, 2, 2, d, None, None, 0.5)
        want, bound = attend_want(q, k, v, torch.ones(b, lk, dtype=torch.bool, device="cuda"), 0.5, element)
        assert_within(o, want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("lq", [1, 130])
def test_cross_attention_without_keys(pkg, element, lq):
    q = normal(gen(0), 2, lq, 2, 64).to(KIND[element])
    o = torch.full_like(q, 5.0)
    pkg.op_cross_attention(q.data_ptr(), None, None, o.data_ptr(), element, 2, lq, 0, 2, 2, 64)
    assert not o.any()


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("lq", [1, 130])
def test_cross_attention_nan_stays_in_its_row(pkg, element, lq):
    """A NaN in a query reaches its own row and head; one in a value its own column; one in a key all rows of its head."""
    q, k, v = (normal(gen(n), 1, l, 2, 64).to(KIND[element]) for n, l in ((0, lq), (1, 300), (2, 300)))
    q[0, 0, 0, 3] = math.nan
    v[0, 7, 1, 5] = math.nan
    o = torch.empty_like(q)
    bad = k.clone()
    for key in (15, 46, 299):
        bad[0, key, 1, 2] = math.nan
        pkg.op_cross_attention(q.data_ptr(), bad.data_ptr(), v.data_ptr(), o.data_ptr(), element, 1, lq, 300, 2, 2, 64)
        assert torch.isnan(o[0, :, 1]).all() and torch.isfinite(o[0, 1:, 0]).all()
        bad[0, key, 1, 2] = 0
    pkg.op_cross_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), element, 1, lq, 300, 2, 2, 64)
    assert torch.isnan(o[0, 0, 0]).all() and torch.isfinite(o[0, 1:, 0]).all()
    assert torch.isnan(o[0, :, 1, 5]).all() and torch.isfinite(o[0, :, 1, :5]).all() and torch.isfinite(o[0, :, 1, 6:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
def test_cross_attention_is_the_same_every_time(pkg, element):
    """The same bits from call to call, and for a sequence of a batch alone, on another stream and in a replayed graph."""
    for lq, lk, heads, kv_heads, d in ((1, 3000, 8, 2, 128), (150, 700, 4, 4, 64)):
        q, k, v = (normal(gen(n), 2, l, h, d).to(KIND[element]) for n, l, h in ((0, lq, heads), (1, lk, kv_heads), (2, lk, kv_heads)))
        o = [torch.empty_like(q) for _ in range(4)]

        def call(to, stream=0):
            pkg.op_cross_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), to.data_ptr(), element, 2, lq, lk, heads, kv_heads, d, stream=stream)

        call(o[0])
        call(o[1])
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        call(o[2], s.cuda_stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(o[3], torch.cuda.current_stream().cuda_stream)
        o[3].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o[0], t) for t in o[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f16", "f32"])
@pytest.mark.parametrize("b,lq,lk,heads,kv_heads,d", [(1, 6, 1399, 16, 2, 128), (1, 64, 600, 8, 8, 64), (2, 100, 777, 4, 4, 160), (1, 700, 513, 2, 1, 96),
                                                      (1, 1, 9000, 2, 2, 64), (1, 20, 5000, 1, 1, 128), (1, 1, 4100, 1, 1, 256), (1, 300, 2000, 1, 1, 200)])
def test_cross_attention_split_keys(pkg, element, b, lq, lk, heads, kv_heads, d):
    """Calls whose keys are cut over warps, CTAs and clusters: with masks, and lengths that leave some of them nothing."""
    mask = torch.rand(b, lk, generator=torch.Generator().manual_seed(lk)) < 0.3
    check_attend(pkg, element, b, lq, lk, heads, kv_heads, d, mask=mask)
    check_attend(pkg, element, b, lq, lk, heads, kv_heads, d, lens=[9] * b)
    check_attend(pkg, element, b, lq, lk, heads, kv_heads, d, lens=[lk - 7] * b, mask=mask)


@pytest.mark.gpu
def test_offsets_past_32_bits(pkg):
    """Rows 2^21 elements apart, 1100 of them: offsets in elements pass 2^31."""
    rows, pitch = 1100, 1 << 21
    for element in ("bf16", "f32"):
        kind = KIND[element]
        big = torch.empty(rows * pitch, device="cuda", dtype=kind)
        view = torch.as_strided(big, (rows, 256), (pitch, 1))
        view.copy_(normal(gen(4), rows, 256))
        size = big.element_size()
        for lq in (1, 200):
            q = normal(gen(5), 1, lq, 1, 128).to(kind)
            o = torch.empty_like(q)
            strides = (lq * 128, 128, 128, 0, pitch, 128, 0, pitch, 128, lq * 128, 128, 128)
            pkg.op_cross_attention(q.data_ptr(), big.data_ptr(), big.data_ptr() + 128 * size, o.data_ptr(), element, 1, lq, rows, 1, 1, 128, strides=strides)
            k, v = view[:, :128].reshape(1, rows, 1, 128), view[:, 128:].reshape(1, rows, 1, 128)
            assert_within(o, *attend_want(q, k, v, torch.ones(1, rows, dtype=torch.bool, device="cuda"), 128 ** -0.5, element))
        y = torch.empty(rows, 256, device="cuda", dtype=kind)
        pkg.op_group_norm(big.data_ptr(), y.data_ptr(), element, 1, rows, 256, 8, None, None, 1e-5, "none", pitch, 0)
        want, off = norm_want(view.reshape(1, rows, 256), 8, None, None, 1e-5, "none")
        assert_within(y.view(1, rows, 256), want, off + U[element] * (want.abs() + off) + TINY[element])
        positions = torch.arange(rows, device="cuda", dtype=torch.int32).view(rows, 1).contiguous()
        want, mag = rotary_want(view.reshape(rows, 2, 128), positions, [64], 10000.0, False, False)
        pkg.op_rotary_axes(big.data_ptr(), big.data_ptr(), element, rows, 2, 128, positions.data_ptr(), [64], strides=(pitch, 128, pitch, 128))
        assert_within(view.reshape(rows, 2, 128), want, 10 * F * mag + U[element] * (want.abs() + 10 * F * mag) + TINY[element])
        del big, view


@pytest.mark.gpu
def test_calls_at_once(pkg):
    """Different calls in flight on several streams, and replays of two captured graphs at once, share nothing."""
    def make(n):
        lq, lk = ((1, 2000), (200, 700), (1500, 60), (40, 900))[n % 4]
        element = ("bf16", "f32")[n // 4]
        q, k, v = (normal(gen(10 * n + i), 2, l, 4, 64).to(KIND[element]) for i, l in enumerate((lq, lk, lk)))
        x = normal(gen(n), 2, 3000 + n, 64).to(KIND[element])
        return element, lq, lk, q, k, v, x, torch.empty_like(q), torch.empty_like(x)

    def run(c, stream):
        element, lq, lk, q, k, v, x, o, y = c
        pkg.op_cross_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), element, 2, lq, lk, 4, 4, 64, stream=stream)
        pkg.op_group_norm(x.data_ptr(), y.data_ptr(), element, 2, x.shape[1], 64, 8, None, None, 1e-5, "swish", stream=stream)

    calls = [make(n) for n in range(8)]
    for c in calls:
        run(c, 0)
    torch.cuda.synchronize()
    alone = [(c[-2].clone(), c[-1].clone()) for c in calls]
    for c in calls:
        c[-2].zero_()
        c[-1].zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        for c, s in zip(calls, streams):
            run(c, s.cuda_stream)
    torch.cuda.synchronize()
    for c, (o, y) in zip(calls, alone):
        assert torch.equal(c[-2], o) and torch.equal(c[-1], y)
    graphs = []
    for c in calls[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(c, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
        c[-2].zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for c, (o, y) in zip(calls[:2], alone):
        assert torch.equal(c[-2], o) and torch.equal(c[-1], y)


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk,heads", [(200, 300, 2), (100, 300, 64), (2000, 100, 16)])
def test_a_wait_that_runs_out_is_reported(pkg, monkeypatch, lq, lk, heads):
    """NCNN_B200_TEST_STALL leaves the first block of keys unloaded and shortens the waits to 2 ms: the call's kernel gives up,
    ncnn_b200_op_check_status says so once, and later calls are right."""
    q, k, v = (normal(gen(n), 1, l, heads, 64).half() for n, l in ((0, lq), (1, lk), (2, lk)))
    o = torch.empty_like(q)

    def call():
        pkg.op_cross_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), "f16", 1, lq, lk, heads, heads, 64)

    pkg.op_check_status()
    monkeypatch.setenv("NCNN_B200_TEST_STALL", "1")
    call()
    monkeypatch.delenv("NCNN_B200_TEST_STALL")
    assert status_of(pkg.op_check_status) == 7
    pkg.op_check_status()
    call()
    pkg.op_check_status()
    assert_within(o, *attend_want(q, k, v, torch.ones(1, lk, dtype=torch.bool, device="cuda"), 0.125, "f16"))


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
def test_a_block_of_an_image_generator(pkg, element):
    """Feature map -> group norm and Swish -> projections to queries, keys and values -> rotary positions of row and column ->
    attention to the image's own tokens -> attention to a text's tokens of ragged lengths, each step against its formula in
    64 bits on the step's own inputs; the whole run also as one captured graph."""
    n, side, c, heads, d, text = 2, 20, 128, 4, 32, 45
    p = side * side
    g = gen(11)
    kind = KIND[element]
    x = (normal(g, n, p, c) + 0.5).to(kind)
    gamma, beta = normal(g, c) * 0.2 + 1, normal(g, c) * 0.2
    w = (normal(g, c, 3 * c) / math.sqrt(c) * 1.5).to(kind)
    states = normal(g, n, text, 2 * c).to(kind)
    lens = torch.tensor([45, 12], dtype=torch.int32, device="cuda")
    grid = torch.stack(torch.meshgrid(torch.arange(side), torch.arange(side), indexing="ij"), -1).view(p, 2).to(torch.int32).cuda().contiguous()
    y, o1, o2 = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    qkv, turned = torch.empty(n, p, 3 * c, device="cuda", dtype=kind), torch.empty(n, p, 2 * c, device="cuda", dtype=kind)
    size = x.element_size()

    def block():
        s = torch.cuda.current_stream().cuda_stream
        pkg.op_group_norm(x.data_ptr(), y.data_ptr(), element, n, p, c, 8, gamma.data_ptr(), beta.data_ptr(), 1e-5, "swish", stream=s)
        torch.matmul(y, w, out=qkv)
        # the queries' and the keys' heads of the projection in one call
        pkg.op_rotary_axes(qkv.data_ptr(), turned.data_ptr(), element, n * p, 2 * heads, d, grid.data_ptr(), [8, 8], 100.0, False, False, p,
                           (3 * c, d, 2 * c, d), stream=s)
        own = (p * 2 * c, 2 * c, d, p * 2 * c, 2 * c, d, p * 3 * c, 3 * c, d, p * c, c, d)
        pkg.op_cross_attention(turned.data_ptr(), turned.data_ptr() + c * size, qkv.data_ptr() + 2 * c * size, o1.data_ptr(), element, n, p, p, heads,
                               heads, d, strides=own, stream=s)
        kv = (p * c, c, d, text * 2 * c, 2 * c, d, text * 2 * c, 2 * c, d, p * c, c, d)
        pkg.op_cross_attention(o1.data_ptr(), states.data_ptr(), states.data_ptr() + c * size, o2.data_ptr(), element, n, p, text, heads, heads, d,
                               lens.data_ptr(), strides=kv, stream=s)

    block()
    torch.cuda.synchronize()
    want, off = norm_want(x, 8, gamma, beta, 1e-5, "swish")
    assert_within(y, want, off + U[element] * (want.abs() + off) + TINY[element])
    want, mag = rotary_want(qkv.view(n * p, 3 * heads, d)[:, : 2 * heads], grid.repeat(n, 1), [8, 8], 100.0, False, False)
    assert_within(turned.view(n * p, 2 * heads, d), want, 10 * F * mag + U[element] * (want.abs() + 10 * F * mag) + TINY[element])
    every = torch.ones(n, p, dtype=torch.bool, device="cuda")
    q, k = (turned[..., i * c:(i + 1) * c].reshape(n, p, heads, d) for i in (0, 1))
    assert_within(o1.view(n, p, heads, d), *attend_want(q, k, qkv[..., 2 * c:].reshape(n, p, heads, d), every, d ** -0.5, element))
    keep = torch.arange(text, device="cuda")[None] < lens[:, None]
    k, v = (states[..., i * c:(i + 1) * c].reshape(n, text, heads, d) for i in (0, 1))
    assert_within(o2.view(n, p, heads, d), *attend_want(o1.view(n, p, heads, d), k, v, keep, d ** -0.5, element))
    first = [t.clone() for t in (y, qkv, turned, o1, o2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block()
    for t in (y, qkv, turned, o1, o2):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for t, was in zip((y, qkv, turned, o1, o2), first):
        assert torch.equal(t, was)
