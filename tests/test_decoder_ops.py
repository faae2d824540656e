"""The operators of a decoder in 8-bit integers, against their formulas in 64 bits: rows quantised, products of tokens, a paged cache
written, read and attended to.

Tolerances follow from the arithmetic.  U[t] is half a step of type t relative to the value (one rounding to it), F = 2^-24 is
fp32's; a sum of n terms in fp32 is off by at most n F times the sum of their magnitudes in any order.  Integers and steps are exact.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}
F = 2.0 ** -24
KIND = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPES = ["f32", "f16", "bf16"]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def assert_within(got, want, bound):
    got = got.double()
    assert int((~torch.isfinite(got)).sum()) == 0
    over = (got - want).abs() - bound
    worst = int(over.argmax())
    assert over.max() <= 0, (float(got.flatten()[worst]), float(want.flatten()[worst]), float(bound.expand_as(want).flatten()[worst]))


def status_of(call):
    with pytest.raises(Exception) as err:
        call()
    return getattr(err.value, "status", type(err.value).__name__)


def host(n=256):
    a = np.zeros(n, np.float32)
    at = a.ctypes.data
    return a, (at + 15) // 16 * 16


# ------------------------------------------------------------------------------------------------ refusals (no GPU)
def test_quantize_rows_refuses(pkg):
    keep = [host() for _ in range(3)]
    x, q, steps = (k[1] for k in keep)

    def call(x=x, q=q, steps=steps, element="f32", rows=2, columns=4, xp=0, qp=0):
        return lambda: pkg.op_quantize_rows(x, element, rows, columns, q, steps, xp, qp)

    assert [status_of(call(**{n: None})) for n in ("x", "q", "steps")] == [1] * 3
    for bad in (dict(rows=-1), dict(columns=0), dict(columns=-4), dict(xp=3), dict(qp=3), dict(q=x), dict(steps=x), dict(steps=q), dict(x=x + 2), dict(steps=steps + 1)):
        assert status_of(call(**bad)) == 2, bad
    assert status_of(call(rows=1 << 40)) == 4 and status_of(call(xp=1 << 50)) == 4
    assert status_of(call(element="i8")) == "ValueError"
    with pytest.raises(pkg.NcnnB200Error, match="device memory"):
        call()()
    call(rows=0)()


def test_inner_product_tokens_refuses(pkg):
    keep = [host() for _ in range(6)]
    x, y, w, ws, bias, space = (k[1] for k in keep)

    def call(x=x, y=y, w=w, ws=ws, space=space, size=1 << 20, element="f32", tokens=2, k=4, n=3, bias=None, act="none", xp=0, yp=0, wp=0):
        return lambda: pkg.op_inner_product_tokens(x, y, element, tokens, k, n, w, ws, space, size, bias, act, xp, yp, wp)

    assert [status_of(call(**{n: None})) for n in ("x", "y", "w", "ws", "space")] == [1] * 5
    for bad in (dict(tokens=-1), dict(k=0), dict(k=131073), dict(n=0), dict(xp=3), dict(yp=2), dict(wp=3), dict(y=x), dict(y=w), dict(y=space), dict(space=x),
                dict(space=space + 4), dict(x=x + 1), dict(ws=ws + 2), dict(bias=bias + 2)):
        assert status_of(call(**bad)) == 2, bad
    assert status_of(call(tokens=1 << 32)) == 4 and status_of(call(wp=1 << 50)) == 4
    assert status_of(call(size=pkg.op_inner_product_tokens_workspace(2, 4) - 1)) == 5
    assert status_of(call(act="cube")) == "ValueError"
    for bad in ((-1, 4), (4, 0), (4, 131073), (1 << 40, 4)):
        assert status_of(lambda: pkg.op_inner_product_tokens_workspace(*bad)) == "ValueError"
    with pytest.raises(pkg.NcnnB200Error, match="device memory"):
        call()()
    call(tokens=0)()


def cache_of(pkg, at, **change):
    v = {**dict(k=at[0], v=at[1], k_steps=at[2], v_steps=at[3], pages=2, page_size=16, kv_heads=2, head_dim=8), **change}
    return pkg.Cache(*(v[n] for n in ("k", "v", "k_steps", "v_steps", "pages", "page_size", "kv_heads", "head_dim")))


def batch_of(pkg, at, **change):
    v = {**dict(table=at[0], lens=at[1], starts=None, sequences=2, tokens=2, table_width=2, max_tokens=0, max_len=0), **change}
    return pkg.CacheBatch(**v)


def test_cache_calls_refuse(pkg):
    keep = [host() for _ in range(9)]
    at = [k[1] for k in keep]
    cache, batch = cache_of(pkg, at), batch_of(pkg, at[4:])
    a, b, space = at[6:]
    calls = {
        "write": lambda c=cache, t=batch, a=a, b=b, element="f32", strides=None: pkg.op_cache_write(c, t, a, b, element, strides),
        "read": lambda c=cache, t=batch, a=a, b=b, element="f32", strides=None: pkg.op_cache_read(c, t, a, b, element, strides),
        "attend": lambda c=cache, t=batch, a=a, b=b, element="f32", strides=None, heads=4, shared=0, scale=0.0:
            pkg.op_cache_attention(c, t, a, b, element, heads, shared, scale, strides, space, 1 << 20),
    }
    for name, call in calls.items():
        for bad in (dict(page_size=8), dict(page_size=24), dict(page_size=2048), dict(head_dim=0), dict(head_dim=257), dict(kv_heads=0), dict(pages=-1),
                    dict(k=at[0] + 8), dict(v_steps=at[3] + 4), dict(v=at[0])):
            assert status_of(lambda: call(c=cache_of(pkg, at, **bad))) == 2, (name, bad)
        for missing in ("k", "v", "k_steps", "v_steps"):
            assert status_of(lambda: call(c=cache_of(pkg, at, **{missing: None}))) == 1
        for bad in (dict(sequences=-1), dict(tokens=-1), dict(tokens=1 << 31), dict(table_width=-1), dict(max_tokens=-1), dict(max_len=-1), dict(max_len=33),
                    dict(lens=at[5] + 2), dict(starts=at[5] + 1)):
            assert status_of(lambda: call(t=batch_of(pkg, at[4:], **bad))) == 2, (name, bad)
        assert status_of(lambda: call(t=batch_of(pkg, at[4:], table_width=1 << 30))) == 4
        assert status_of(lambda: call(t=batch_of(pkg, at[4:], table=None))) == 1 and status_of(lambda: call(t=batch_of(pkg, at[4:], lens=None))) == 1
        assert status_of(lambda: call(a=None)) == 1 or name == "read"
        assert status_of(lambda: call(a=a + 2)) == 2 and status_of(lambda: call(b=b + 2)) == 2
        assert status_of(lambda: call(b=at[0])) == 2
        assert status_of(lambda: call(strides=(-16, 8, 16, 8))) == 2 and status_of(lambda: call(strides=(1 << 60, 8, 16, 8))) == 4
        assert status_of(lambda: call(strides=(16, 8))) == "ValueError" and status_of(lambda: call(element="i8")) == "ValueError"
        with pytest.raises(pkg.NcnnB200Error, match="device memory"):
            call()
        call(t=batch_of(pkg, at[4:], tokens=0))
        call(t=batch_of(pkg, at[4:], sequences=0))
    assert status_of(lambda: calls["read"](a=None, b=None)) == 1 and status_of(lambda: calls["read"](a=a, b=a)) == 2
    assert status_of(lambda: calls["read"](strides=(16, 7, 16, 8))) == 2
    assert status_of(lambda: calls["attend"](strides=(32, 8, 24, 8))) == 2
    for bad in (dict(heads=0), dict(heads=3), dict(shared=-16), dict(shared=8), dict(shared=48), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(b=a)):
        assert status_of(lambda: calls["attend"](**bad)) == 2, bad
    for bad in (dict(heads=3), dict(shared=8)):
        assert status_of(lambda: pkg.op_cache_attention_workspace(cache, batch, **{**dict(heads=4, shared=0), **bad})) == "ValueError"
    assert pkg.op_cache_attention_workspace(cache, batch_of(pkg, at[4:], tokens=0), 4) == 0


# ------------------------------------------------------------------------------------------------ rows to integers
def quantised(x):
    """Integers and steps of rows, by the definition: whole numbers of halves in 64 bits, which are exact (126 x at most 2^-33 off)."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    live = (top >= 2.0 ** -100) & torch.isfinite(top)
    halves = torch.floor(254 * x.abs() / torch.where(live, top, 1.0))
    q = torch.where(live, torch.sign(x) * torch.floor((halves + 1) / 2), 0.0)
    step = torch.where(live, top / 127, torch.where(torch.isfinite(top), 0.0, math.nan))
    return torch.nan_to_num(q).to(torch.int8), step[..., 0].float()


def same_steps(got, want):
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def check_rows(pkg, x, element, pitch=0, shift=0):
    rows, columns = x.shape
    xp = x.stride(0) if rows > 1 else columns
    qp = pitch or columns
    q = torch.full((rows * qp + shift,), 99, dtype=torch.int8, device="cuda")
    steps = torch.full((rows,), -1.0, device="cuda")
    pkg.op_quantize_rows(x.data_ptr(), element, rows, columns, q.data_ptr() + shift, steps.data_ptr(), xp, qp)
    torch.cuda.synchronize()
    want, want_steps = quantised(x)
    got = torch.as_strided(q, (rows, columns), (qp, 1), shift)
    assert torch.equal(got, want)
    same_steps(steps, want_steps)
    if qp > columns:  # what lies between the rows is not touched
        assert bool((torch.as_strided(q, (rows - 1, qp - columns), (qp, 1), shift + columns) == 99).all())


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 8), (3, 7), (1, 4096), (64, 4096), (5, 4099), (2000, 128), (1500, 1000), (2, 40000), (1024, 513), (1, 131072)])
def test_quantize_rows(pkg, element, rows, columns):
    g = gen(rows + columns)
    check_rows(pkg, (normal(g, rows, columns) * normal(g, columns).abs()).to(KIND[element]), element)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
def test_quantize_rows_layouts(pkg, element):
    g = gen(3)
    wide = normal(g, 9, 200).to(KIND[element])
    for columns, at, pitch, shift in ((64, 0, 64, 0), (64, 8, 80, 16), (64, 3, 64, 0), (61, 1, 67, 5), (64, 8, 72, 4), (128, 16, 131, 1)):
        check_rows(pkg, wide[:, at:at + columns], element, pitch, shift)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
def test_quantize_rows_halves_and_ends(pkg, element):
    kind = KIND[element]
    # every multiple of a half below 127: halves go away from zero
    halves = torch.arange(-254, 255, device="cuda") / 2
    rows = [halves * f for f in (1.0, 2.0 ** -14 if element == "f16" else 2.0 ** -90, 2.0 ** 8 if element == "f16" else 2.0 ** 100, 0.75 if element == "f32" else 1.0)]
    info = torch.finfo(kind)
    rows += [torch.full_like(halves, info.max), torch.full_like(halves, -info.max), torch.linspace(-1, 1, halves.numel(), device="cuda") * info.max]
    rows += [torch.zeros_like(halves), torch.full_like(halves, info.tiny if element != "f16" else 0.0)]
    for bad in (math.nan, math.inf, -math.inf):
        row = halves.clone()
        row[17] = bad
        rows.append(row)
    check_rows(pkg, torch.stack(rows).to(kind), element)


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f16", "bf16"])
def test_quantize_rows_every_pair_of_numbers(pkg, element):
    """Rows of all positive numbers of an octave under each largest one of the octaves above: every quotient that there is, ties among them."""
    bits = 10 if element == "f16" else 7
    mantissa = 1 + torch.arange(2 ** bits, device="cuda") / 2 ** bits
    x = torch.cat([mantissa * 2.0 ** -e for e in range(8)])
    for tops in mantissa.split(128):
        rows = x.repeat(tops.numel(), 1)
        check_rows(pkg, torch.cat((torch.minimum(rows, tops[:, None]), tops[:, None]), 1).to(KIND[element]), element)


# ------------------------------------------------------------------------------------------------ products of tokens
def product_want(q, steps, w, weight_steps, bias, act, element):
    """The result and how far the roundings may take it: the sum's to fp32, the steps' product and its product with the sum (3 F of it),
    the fma's; an activation's slope is below 1.13; then its own error and the rounding to the type."""
    t = (q.double() @ w.double().T) * steps.double()[:, None] * weight_steps.double()
    off = 3.01 * F * t.abs()
    if bias is not None:
        t = t + bias.double()
    off = off + F * t.abs()
    if act == "relu":
        y, off = torch.relu(t), off
    elif act == "swish":
        y = t * torch.sigmoid(t)
        # 16 bits: __expf is off by 2 + 1.173 |t| steps of 2 F, __fdividef by 2, the sum by 1/2; fp32: expf by 1, and two roundings.
        # Below -87 the quotient may be flushed: 2^-120 bounds what is lost.
        off = 1.13 * off + y.abs() * 2 * F * ((5 + 1.2 * t.abs()) if element != "f32" else 4) + 2.0 ** -118
    elif act == "gelu":
        y = t * torch.special.ndtr(t)
        # erfcf is off by 4 steps; its argument's two roundings count 2 z^2 + 2 times (z = t / sqrt 2: t^2 + 2)
        # 16 bits: a fit of erfcx that is off by 2^-16.8, times an exponential of z^2 (which is F off, so the power z^2 F) by __expf, 2 +
        # 1.173 z^2 steps of 2 F, and a quotient by 2 steps
        own = F * (12 + 3 * (t.clamp_max(0) ** 2 + 2)) if element == "f32" else 2.0 ** -16.8 + F * (16 + 2 * t ** 2).clamp_max(2.0 ** 10)
        off = 1.13 * off + y.abs() * own + 2.0 ** -118
    else:
        y = t
    return y, off + U[element] * (y.abs() + off) + TINY[element]


def check_product(pkg, element, m, k, n, act="none", bias=True, x_pitch=0, y_pitch=0, w_pitch=0, shift=0, w_shift=0, seed=0, extreme=False):
    g = gen(seed + m + k + n)
    xp, yp, wp = x_pitch or k, y_pitch or n, w_pitch or k
    x = torch.empty(m * xp + shift, device="cuda", dtype=KIND[element]).copy_(normal(g, m * xp + shift))
    w = torch.randint(-127, 128, (n * wp + w_shift,), generator=g, device="cuda", dtype=torch.int8)
    y = torch.full((m * yp + shift,), 5.0, device="cuda", dtype=KIND[element])
    if extreme:  # the largest sums that there are
        x.fill_(1.0)
        w.fill_(127)
        w[:wp] = -127
    ws = (normal(g, n).abs() + 0.2) / (40 * math.sqrt(k)) if not extreme else torch.full((n,), 1.0 / (127 * k), device="cuda")
    b = normal(g, n) if bias else None
    space = torch.empty(pkg.op_inner_product_tokens_workspace(m, k), dtype=torch.uint8, device="cuda")
    size = KIND[element].itemsize
    pkg.op_inner_product_tokens(x.data_ptr() + shift * size, y.data_ptr() + shift * size, element, m, k, n, w.data_ptr() + w_shift, ws.data_ptr(),
                                space.data_ptr(), space.numel(), None if b is None else b.data_ptr(), act, xp, yp, wp)
    torch.cuda.synchronize()
    xv, yv = (torch.as_strided(t, (m, e), (p, 1), shift) for t, e, p in ((x, k, xp), (y, n, yp)))
    q, steps = quantised(xv)
    want, bound = product_want(q, steps, torch.as_strided(w, (n, k), (wp, 1), w_shift), ws, b, act, element)
    assert_within(yv, want, bound)
    if yp > n and m > 1:
        assert bool((torch.as_strided(y, (m - 1, yp - n), (yp, 1), shift + n) == 5.0).all())
    return yv


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("m,k,n,act", [(1, 1, 1, "none"), (1, 64, 128, "relu"), (1, 4096, 512, "none"), (2, 16, 40, "swish"), (3, 1000, 129, "gelu"),
                                       (16, 256, 256, "none"), (17, 272, 300, "none"), (33, 4096, 1000, "swish"), (64, 512, 2048, "relu"),
                                       (100, 48, 33, "gelu"), (128, 128, 128, "none"), (129, 2064, 257, "none"), (200, 640, 384, "swish"),
                                       (257, 1024, 512, "none"), (300, 4112, 100, "gelu"), (513, 144, 1040, "none"), (1000, 2048, 1000, "relu")])
def test_inner_product_tokens(pkg, element, m, k, n, act):
    check_product(pkg, element, m, k, n, act, bias=(m + n) % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_inner_product_tokens_layouts(pkg, element, m):
    check_product(pkg, element, m, 96, 80, "swish", x_pitch=104, y_pitch=88, w_pitch=112)
    check_product(pkg, element, m, 100, 81, "none", x_pitch=101, y_pitch=83, w_pitch=112)
    check_product(pkg, element, m, 100, 82, "none", shift=1)
    check_product(pkg, element, m, 128, 64, "relu", shift=3, w_shift=16)
    check_product(pkg, element, m, 128, 64, "none", w_shift=5, w_pitch=131)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(1, 40), (300, 40), (70, 300)])
def test_inner_product_tokens_largest_sums(pkg, m, n):
    check_product(pkg, "f32", m, 131072, n, extreme=True)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 20, 300])
def test_inner_product_tokens_nonfinite(pkg, m):
    """A token with a NaN or an infinity is NaN, and no other is."""
    g = gen(m)
    k, n = 128, 96
    x = normal(g, m, k)
    x[m // 2, 3] = math.inf
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    ws = normal(g, n).abs()
    space = torch.empty(pkg.op_inner_product_tokens_workspace(m, k), dtype=torch.uint8, device="cuda")
    for act in ("none", "relu", "swish", "gelu"):
        y = torch.zeros(m, n, device="cuda")
        pkg.op_inner_product_tokens(x.data_ptr(), y.data_ptr(), "f32", m, k, n, w.data_ptr(), ws.data_ptr(), space.data_ptr(), space.numel(), activation=act)
        torch.cuda.synchronize()
        bad = torch.isnan(y).any(1)
        assert bool(torch.isnan(y[m // 2]).all()) and int(bad.sum()) == 1


# ------------------------------------------------------------------------------------------------ the cache
class Setup:
    """A cache whose pages lie in any order, sequences of given lengths and numbers of new tokens.  What no token has been written to
    holds integers of any size and steps of NaN."""

    def __init__(self, pkg, new, lens, kv_heads, d, page, shared=0, starts=True, spare=2, behind=0, seed=0, fill=True, max_tokens=None, max_len=None, lead=0):
        g = gen(seed)
        self.new, self.lens, self.page, self.d, self.kv_heads, self.shared = new, lens, page, d, kv_heads, shared
        b, self.row = len(lens), (d + 15) // 16 * 16
        self.width = max(1, (max(lens) + page - 1) // page)
        need = shared // page + sum(max(0, (n + page - 1) // page - shared // page) for n in lens)
        self.pages = need + spare
        order = torch.randperm(self.pages, generator=g, device="cuda", dtype=torch.int32)
        self.table = torch.full((b, self.width), -7, dtype=torch.int32, device="cuda")
        used = shared // page
        self.table[0, :used] = order[:used]
        own = torch.full((b, self.width), -7, dtype=torch.int32, device="cuda")
        for i, n in enumerate(lens):
            count = max(0, (n + page - 1) // page - shared // page)
            self.table[i, shared // page:shared // page + count] = order[used:used + count]
            used += count
        self.whole = self.table.clone()  # every sequence's own pages and the shared ones
        self.whole[:, :shared // page] = self.table[0, :shared // page]
        self.ints, self.steps = {}, {}
        for name in "kv":
            self.ints[name] = torch.randint(-128, 128, (self.pages, kv_heads, page, self.row), generator=g, device="cuda", dtype=torch.int8)
            self.steps[name] = torch.full((self.pages, kv_heads, page), math.nan, device="cuda")
        self.len_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
        firsts = [lead]
        for n in new:
            firsts.append(firsts[-1] + n)
        self.firsts, self.tokens = firsts, firsts[-1] + behind
        self.starts = torch.tensor(firsts, dtype=torch.int32, device="cuda") if starts else None
        if fill:
            for i, n in enumerate(lens):
                for p in range((n + page - 1) // page):
                    at = int(self.whole[i, p])
                    if at < 0 or at >= self.pages:
                        continue
                    rows = min(page, n - p * page)
                    for name in "kv":
                        self.ints[name][at, :, :rows] = torch.randint(-127, 128, (kv_heads, rows, self.row), generator=g, device="cuda", dtype=torch.int8)
                        self.steps[name][at, :, :rows] = (normal(g, kv_heads, rows).abs() + 0.3) / 70
        self.cache = pkg.Cache(self.ints["k"].data_ptr(), self.ints["v"].data_ptr(), self.steps["k"].data_ptr(), self.steps["v"].data_ptr(), self.pages, page,
                               kv_heads, d)
        self.batch = pkg.CacheBatch(self.table.data_ptr(), self.len_t.data_ptr(), None if self.starts is None else self.starts.data_ptr(), b, self.tokens,
                                    self.width, max(new + [0]) if max_tokens is None else max_tokens, max(lens) if max_len is None else max_len)

    def held(self, name, i, length):
        """A sequence's values in 64 bits [kv_heads][length][d], and which of its positions are there."""
        pages = self.whole[i, :(length + self.page - 1) // self.page].long()
        there = (pages >= 0) & (pages < self.pages)
        at = torch.where(there, pages, 0)
        x = self.ints[name][at][..., :self.d].double() * self.steps[name][at].double()[..., None]
        x = x.permute(1, 0, 2, 3).reshape(self.kv_heads, -1, self.d)[:, :length]
        return x, there.repeat_interleave(self.page)[:length]


def strided(g, kind, tokens, heads, d, strides, shift):
    ts, hs = strides or (heads * d, d)
    buf = normal(g, max(0, tokens - 1) * ts + (heads - 1) * hs + d + shift).to(kind)
    return buf, torch.as_strided(buf, (tokens, heads, d), (ts, hs, 1), shift)


def check_write_read(pkg, element, s, strides=None, shift=0, seed=0):
    g = gen(seed + 1)
    kind, size = KIND[element], KIND[element].itemsize
    four = None if strides is None else (*strides, *strides)
    src = {n: strided(g, kind, s.tokens, s.kv_heads, s.d, strides, shift) for n in "kv"}
    want_i = {n: s.ints[n].clone() for n in "kv"}
    want_s = {n: s.steps[n].clone() for n in "kv"}
    places = []
    for i, count in enumerate(s.new):
        for j in range(count):
            p = s.lens[i] - count + j
            page = int(s.whole[i, p // s.page]) if p >= 0 else -1
            places.append((s.firsts[i] + j, page if 0 <= page < s.pages else -1, p % s.page))
    ok = [(t, page, at) for t, page, at in places if page >= 0]
    if ok:
        t, page, at = (torch.tensor(c, device="cuda") for c in zip(*ok))
        for n in "kv":
            q, steps = quantised(src[n][1][t])
            want_i[n][page, :, at] = torch.nn.functional.pad(q, (0, s.row - s.d))
            want_s[n][page, :, at] = steps
    pkg.op_cache_write(s.cache, s.batch, src["k"][0].data_ptr() + shift * size, src["v"][0].data_ptr() + shift * size, element, four)
    torch.cuda.synchronize()
    for n in "kv":
        assert torch.equal(s.ints[n], want_i[n])
        same_steps(s.steps[n], want_s[n])
    out = {n: strided(g, kind, s.tokens, s.kv_heads, s.d, strides, shift) for n in "kv"}
    before = {n: out[n][0].clone() for n in "kv"}
    pkg.op_cache_read(s.cache, s.batch, out["k"][0].data_ptr() + shift * size, out["v"][0].data_ptr() + shift * size, element, four)
    torch.cuda.synchronize()
    for n in "kv":
        # one product in fp32 and one rounding to the type: what torch does, bit for bit
        want = before[n].clone()
        view = torch.as_strided(want, out[n][1].shape, out[n][1].stride(), shift)
        for t, page, at in places:
            view[t] = (s.ints[n][page, :, at, :s.d].float() * s.steps[n][page, :, at][:, None]).to(kind) if page >= 0 else 0.0
        assert torch.equal(torch.nan_to_num(out[n][0], nan=77.0), torch.nan_to_num(want, nan=77.0))
        alone = before[n].clone()
        pkg.op_cache_read(s.cache, s.batch, *(alone.data_ptr() + shift * size if x == n else None for x in "kv"), element, four)
        torch.cuda.synchronize()
        assert torch.equal(torch.nan_to_num(alone, nan=77.0), torch.nan_to_num(want, nan=77.0))


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("new,lens,kv_heads,d,page", [([1], [1], 1, 1, 16), ([1, 1, 1], [1, 16, 17], 2, 64, 16), ([3, 0, 5, 1], [3, 7, 40, 1], 3, 72, 16),
                                                      ([33, 2], [100, 2], 8, 128, 32), ([4, 4], [70, 2], 2, 256, 64), ([1, 3], [5, 3], 1, 40, 128),
                                                      ([2, 2, 2], [1, 0, 3], 2, 23, 16), ([17, 1], [1024, 1], 1, 200, 1024)])
def test_cache_write_and_read(pkg, element, new, lens, kv_heads, d, page):
    s = Setup(pkg, new, lens, kv_heads, d, page, fill=False, starts=any(n != 1 for n in new))
    check_write_read(pkg, element, s)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
def test_cache_layouts_and_rows_without_a_place(pkg, element):
    for d, strides, shift in ((64, (400, 72), 0), (64, (401, 65), 0), (64, (64, 1024), 8), (48, None, 1), (30, (200, 31), 3)):
        check_write_read(pkg, element, Setup(pkg, [2, 0, 7], [2, 9, 50], 3, d, 16, behind=4, lead=2, fill=False), strides, shift)
    # pages that are not there
    s = Setup(pkg, [20, 5], [40, 5], 2, 64, 16, fill=False)
    for bad in (-1, s.pages, 1 << 30, -(1 << 31)):
        s.whole[0, 1] = s.table[0, 1] = bad
        check_write_read(pkg, element, s)
    # tokens above max_tokens are left alone, lengths are held to max_len
    s = Setup(pkg, [20, 5], [40, 5], 2, 64, 16, fill=False, max_tokens=6)
    g = gen(5)
    x = normal(g, s.tokens, 2, 64).to(KIND[element])
    before = {n: s.ints[n].clone() for n in "kv"}
    pkg.op_cache_write(s.cache, s.batch, x.data_ptr(), x.data_ptr(), element)
    torch.cuda.synchronize()
    changed = {(p, at) for p, at in (s.ints["k"] != before["k"]).any(-1).any(1).nonzero().tolist()}
    want = {(int(s.table[0, p // 16]), p % 16) for p in range(20, 26)} | {(int(s.table[1, 0]), p) for p in range(5)}
    assert changed == want


# ------------------------------------------------------------------------------------------------ attention over the cache
def cache_attend_want(s, q, scale, element):
    """The result and its tolerance, token by token of each sequence.

    A score: d products summed in fp32 (truncated sums may lose 2 F a term), the steps and the scale 8 F of the sizes; a probability is
    off by as much, the sum over the keys by 2 n F and the exponential and the factors of joined ranges by 16 F.  Products with values
    take the probabilities in terms of bf16: 2^-17 of each where there are two, 2^-26 with three; 16-bit queries of many rows
    round them once to bf16 (2^-8).  What is below fp32's smallest normal number may be taken for zero: probabilities under 2^-126 of the
    row's largest, whose n keys would have added 2^-126 |v| each to a result over a sum of 1 or more (a key of weight 1 whose value is
    exactly 0 leaves nothing else to see), and products of a probability and a step, which an integer of at most 127 multiplies."""
    heads = q.shape[1]
    group = heads // s.kv_heads
    o, bound = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    terms = {"f32": 2.0 ** -25, "f16": 2.0 ** -16, "bf16": 2.0 ** -8}[element]
    for i, count in enumerate(s.new):
        length = s.lens[i]
        if count == 0 or length == 0:
            continue
        k, there = s.held("k", i, length)
        v, _ = s.held("v", i, length)
        position = torch.arange(length - count, length, device="cuda")
        see = (torch.arange(length, device="cuda")[None] <= position[:, None]) & there[None]
        any_key = see.any(1)
        rows = slice(s.firsts[i], s.firsts[i] + count)
        for h in range(heads):
            kk, vv = torch.nan_to_num(k[h // group]), torch.nan_to_num(v[h // group])
            qq = q[rows, h].double()
            sc = qq @ kk.T * scale
            p = torch.softmax(sc.masked_fill(~see, -math.inf), -1)
            p = torch.where(any_key[:, None], p, 0.0)
            oo, spread = p @ vv, p @ vv.abs()
            ds = (2 * s.d + 8) * F * ((qq.abs() @ kk.abs().T) * scale).amax(-1, keepdim=True) + 8 * F * sc.abs().amax(-1, keepdim=True)
            rel = 2 * ds + 4 * length * F + 24 * F + terms
            o[rows, h] = oo
            lost = 2.0 ** -126 * length * (vv.abs().amax() + 127)
            bound[rows, h] = rel * spread + lost + U[element] * (oo.abs() + rel * spread) + TINY[element]
    return o, bound


def attend(pkg, s, q, o, element, heads, shared=0, scale=0.0, strides=None, stream=0, space=None):
    if space is None:
        space = torch.empty(max(16, pkg.op_cache_attention_workspace(s.cache, s.batch, heads, shared)), dtype=torch.uint8, device="cuda")
        space.fill_(255)  # (NaN: nothing is read that has not been written)
    pkg.op_cache_attention(s.cache, s.batch, q.data_ptr(), o.data_ptr(), element, heads, shared, scale, strides, space.data_ptr(), space.numel(), stream)
    return space


def check_attention(pkg, element, s, heads, shared=0, scale=0.0, strides=None, shift=0, spread=1.0, seed=0):
    g = gen(seed + 2)
    kind, size = KIND[element], KIND[element].itemsize
    qb, q = strided(g, kind, s.tokens, heads, s.d, None if strides is None else strides[:2], shift)
    q.mul_(spread)
    ob, o = strided(g, kind, s.tokens, heads, s.d, None if strides is None else strides[2:], shift)
    before = ob.clone()
    attend(pkg, s, qb[shift:], ob[shift:], element, heads, shared, scale, strides)
    pkg.op_check_status()
    want, bound = cache_attend_want(s, q, scale or 1 / math.sqrt(s.d), element)
    rows = slice(s.firsts[0], s.firsts[-1])
    assert_within(o[rows], want[rows], bound[rows])
    # everything else is as it was
    whole = before.clone()
    torch.as_strided(whole, o.shape, o.stride(), shift)[rows] = o[rows]
    assert torch.equal(torch.nan_to_num(whole), torch.nan_to_num(ob))
    return o


SHAPES = [([1], [1], 1, 1, 64, 16), ([1], [4097], 32, 8, 128, 16), ([1, 1, 1], [1, 16, 900], 4, 4, 64, 16), ([1] * 9, [0, 1, 15, 16, 17, 127, 128, 129, 700], 8, 1, 128, 32),
          ([3, 0, 5, 1], [3, 7, 340, 1], 6, 3, 72, 16), ([8, 2], [1100, 2], 14, 2, 80, 64), ([1, 1], [333, 50], 5, 5, 40, 16), ([1, 4], [2500, 90], 4, 2, 256, 128),
          ([70, 1, 33], [70, 500, 333], 8, 2, 128, 16), ([150, 20], [400, 20], 4, 4, 64, 32), ([260], [260], 2, 1, 96, 16), ([300, 40], [1300, 77], 16, 2, 128, 64),
          ([2, 2, 2], [1, 0, 3], 2, 2, 33, 16), ([600], [2000], 3, 3, 128, 16), ([131, 7], [131, 300], 7, 1, 64, 16), ([64] * 5, [64, 200, 1000, 65, 128], 10, 2, 112, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("new,lens,heads,kv_heads,d,page", SHAPES)
def test_cache_attention(pkg, element, new, lens, heads, kv_heads, d, page):
    s = Setup(pkg, new, lens, kv_heads, d, page, starts=any(n != 1 for n in new))
    check_attention(pkg, element, s, heads)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("new,lens,shared,heads,kv_heads,d,page", [
    ([1] * 12, [97, 96, 200, 130, 111, 97, 98, 99, 100, 101, 102, 400], 96, 8, 2, 128, 16), ([1, 1], [2049, 2100], 2048, 4, 1, 64, 64),
    ([1] * 40, [1030 + 7 * i for i in range(40)], 1024, 32, 8, 128, 32), ([5, 3, 9], [21, 100, 70], 16, 6, 3, 72, 16),
    ([30, 1], [30, 64], 64, 4, 2, 64, 32), ([100, 50, 80], [700, 562, 900], 512, 8, 2, 128, 128), ([1] * 3, [10, 300, 64], 256, 4, 4, 256, 64),
    ([1], [5000], 4096, 16, 2, 128, 16)])
def test_cache_attention_shared_prefix(pkg, element, new, lens, shared, heads, kv_heads, d, page):
    s = Setup(pkg, new, lens, kv_heads, d, page, shared=shared, starts=any(n != 1 for n in new))
    check_attention(pkg, element, s, heads, shared)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("count", [1, 3, 140])
def test_cache_attention_layouts(pkg, element, count):
    for strides, d, shift in (((600, 72, 640, 80), 64, 0), ((600, 72, 640, 80), 64, 8), ((601, 75, 333, 65), 64, 1), ((64, 64 * 300, 128, 128 * 300), 64, 0), (None, 50, 1)):
        s = Setup(pkg, [count, 0, count], [count, 9, 400], 2, d, 16, behind=3, lead=2)
        check_attention(pkg, element, s, 4, strides=strides, shift=shift)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("count", [1, 5, 150])
def test_cache_attention_pages_that_are_not_there(pkg, element, count):
    for bad in (-1, 1 << 30, -(1 << 31)):
        s = Setup(pkg, [count, count], [500, 200], 2, 128, 16, spare=3)
        for i, p in ((0, 3), (0, 11), (0, 31), (1, 0)):
            s.whole[i, p] = s.table[i, p] = bad
        check_attention(pkg, element, s, 8)
    s = Setup(pkg, [count], [count], 2, 128, 16, spare=3)
    s.whole[:] = s.table[:] = -1
    assert not bool(check_attention(pkg, element, s, 8).any())


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("count", [1, 150])
def test_cache_attention_scores(pkg, element, count):
    s = Setup(pkg, [count, count], [900, 200], 2, 64, 16)
    check_attention(pkg, element, s, 4, scale=0.7)
    check_attention(pkg, element, s, 4, scale=1e-6)
    check_attention(pkg, element, s, 4, spread=30.0)
    # values of tokens far from one another in size
    for name in "kv":
        far = 2.0 ** torch.randint(-40, 12, s.steps[name].shape, generator=gen(4), device="cuda")
        s.steps[name].mul_(far if name == "v" else 1.0)
    check_attention(pkg, element, s, 4, spread=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("count", [2, 150])
def test_cache_attention_nan_reaches_only_who_sees_it(pkg, element, count):
    s = Setup(pkg, [count, count], [300, 200], 2, 128, 16)
    place = 300 - count + 1  # the second new token's position
    page, at = int(s.table[0, place // 16]), place % 16
    for name in "kv":
        kept = s.steps[name][page, 1, at].clone()
        s.steps[name][page, 1, at] = math.nan
        q = normal(gen(9), s.tokens, 8, 128).to(KIND[element])
        o = torch.zeros_like(q)
        attend(pkg, s, q, o, element, 8)
        pkg.op_check_status()
        bad = torch.isnan(o).any(-1)
        assert bool(bad[1:count, 4:].all()) and not bool(bad[:1].any()) and not bool(bad[:, :4].any()) and not bool(bad[count:].any())
        s.steps[name][page, 1, at] = kept


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("count,shared", [(1, 0), (1, 512), (100, 0), (100, 512)])
def test_cache_attention_is_the_same_every_time(pkg, element, count, shared):
    s = Setup(pkg, [count] * 3, [600 + count, 700 + count, 512 + count], 2, 128, 16, shared=shared)
    q = normal(gen(9), s.tokens, 8, 128).to(KIND[element])
    got = []
    for _ in range(3):
        o = torch.zeros_like(q)
        attend(pkg, s, q, o, element, 8, shared)
        pkg.op_check_status()
        got.append(o)
    assert all(torch.equal(got[0], x) for x in got)


@pytest.mark.gpu
def test_offsets_past_32_bits(pkg):
    """A cache of more than 2^32 bytes of keys, the last pages in use."""
    kv_heads, d, page = 8, 128, 16
    pages = (1 << 32) // (kv_heads * d * page) + 40
    if torch.cuda.mem_get_info()[0] < 3 * pages * kv_heads * d * page:
        pytest.skip("not enough device memory")
    ints = [torch.zeros(pages, kv_heads, page, d, dtype=torch.int8, device="cuda") for _ in "kv"]
    steps = [torch.zeros(pages, kv_heads, page, device="cuda") for _ in "kv"]
    cache = pkg.Cache(*(t.data_ptr() for t in ints + steps), pages, page, kv_heads, d)
    count = 300
    for heads in (8, 32):
        table = torch.arange(pages - 1, pages - 31, -1, device="cuda", dtype=torch.int32)[None].contiguous()
        lens = torch.tensor([count], dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, count], dtype=torch.int32, device="cuda")
        batch = pkg.CacheBatch(table.data_ptr(), lens.data_ptr(), starts.data_ptr(), 1, count, 30)
        g = gen(1)
        k, v, q = normal(g, count, kv_heads, d).bfloat16(), normal(g, count, kv_heads, d).bfloat16(), normal(g, count, heads, d).bfloat16()
        pkg.op_cache_write(cache, batch, k.data_ptr(), v.data_ptr(), "bf16")
        back = torch.zeros_like(k)
        pkg.op_cache_read(cache, batch, back.data_ptr(), None, "bf16")
        o = torch.zeros_like(q)
        space = torch.empty(max(16, pkg.op_cache_attention_workspace(cache, batch, heads)), dtype=torch.uint8, device="cuda")
        pkg.op_cache_attention(cache, batch, q.data_ptr(), o.data_ptr(), "bf16", heads, workspace_ptr=space.data_ptr(), workspace_bytes=space.numel())
        pkg.op_check_status()
        kd, vd = ((i.double() * st.double()[..., None]) for i, st in (quantised(k), quantised(v)))
        assert torch.equal(back, kd.float().bfloat16()) or float((back.double() - kd).abs().max()) <= U["bf16"] * 1.01 * float(kd.abs().max())
        for h in (0, heads - 1):
            sc = (q[:, h].double() @ kd[:, h * 8 // heads].T / math.sqrt(d)).masked_fill(torch.ones(count, count, device="cuda").triu(1).bool(), -math.inf)
            want = torch.softmax(sc, -1) @ vd[:, h * 8 // heads]
            spread = torch.softmax(sc, -1) @ vd[:, h * 8 // heads].abs()
            assert_within(o[:, h], want, 3 * U["bf16"] * spread)
        del table
    assert int(ints[0][:pages - 31].abs().max()) == 0


# ------------------------------------------------------------------------------------------------ together
def decoder_step(pkg, w, s, x, heads, kv_heads, d, positions, space, qkv, turned, o, y, stream=0):
    """Joint projection, rotary positions, keys and values into the cache, attention, projection back."""
    tokens, width = x.shape
    joint = (heads + 2 * kv_heads) * d
    pkg.op_inner_product_tokens(x.data_ptr(), qkv.data_ptr(), "bf16", tokens, width, joint, w["in"].data_ptr(), w["in_steps"].data_ptr(),
                                space[0].data_ptr(), space[0].numel(), stream=stream)
    size = 2
    pkg.op_rotary_axes(qkv.data_ptr(), turned.data_ptr(), "bf16", tokens, heads + kv_heads, d, positions.data_ptr(), [d // 2],
                       strides=(joint, d, (heads + kv_heads) * d, d), stream=stream)
    pkg.op_cache_write(s.cache, s.batch, turned.data_ptr() + heads * d * size, qkv.data_ptr() + (heads + kv_heads) * d * size, "bf16",
                       ((heads + kv_heads) * d, d, joint, d), stream=stream)
    pkg.op_cache_attention(s.cache, s.batch, turned.data_ptr(), o.data_ptr(), "bf16", heads, strides=((heads + kv_heads) * d, d, heads * d, d),
                           workspace_ptr=space[1].data_ptr(), workspace_bytes=space[1].numel(), stream=stream)
    pkg.op_inner_product_tokens(o.data_ptr(), y.data_ptr(), "bf16", tokens, heads * d, width, w["out"].data_ptr(), w["out_steps"].data_ptr(),
                                space[0].data_ptr(), space[0].numel(), stream=stream)


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 40])
def test_a_decoder_step(pkg, count):
    """A run of them as a decoder makes it, eager and captured: each operator's output against its formula on what it was given."""
    heads, kv_heads, d, width = 8, 2, 64, 256
    joint = (heads + 2 * kv_heads) * d
    s = Setup(pkg, [count] * 3, [count, 100 + count, 33 + count], kv_heads, d, 16)
    g = gen(11)
    w = {}
    for name, rows, columns in (("in", joint, width), ("out", width, heads * d)):
        full = normal(g, rows, columns) / math.sqrt(columns)
        w[name] = torch.empty(rows, columns, dtype=torch.int8, device="cuda")
        w[name + "_steps"] = torch.empty(rows, device="cuda")
        pkg.op_quantize_rows(full.data_ptr(), "f32", rows, columns, w[name].data_ptr(), w[name + "_steps"].data_ptr())
    x = normal(g, s.tokens, width).bfloat16()
    positions = torch.cat([torch.arange(n - count, n, device="cuda", dtype=torch.int32) for n in s.lens])[:, None].contiguous()
    space = [torch.empty(pkg.op_inner_product_tokens_workspace(s.tokens, max(width, heads * d)), dtype=torch.uint8, device="cuda"),
             torch.empty(max(16, pkg.op_cache_attention_workspace(s.cache, s.batch, heads)), dtype=torch.uint8, device="cuda")]
    qkv = torch.zeros(s.tokens, joint, device="cuda", dtype=torch.bfloat16)
    turned = torch.zeros(s.tokens, heads + kv_heads, d, device="cuda", dtype=torch.bfloat16)
    o = torch.zeros(s.tokens, heads, d, device="cuda", dtype=torch.bfloat16)
    y = torch.zeros(s.tokens, width, device="cuda", dtype=torch.bfloat16)
    args = (pkg, w, s, x, heads, kv_heads, d, positions, space, qkv, turned, o, y)
    decoder_step(*args)
    pkg.op_check_status()

    def check():
        want, bound = product_want(*quantised(x), w["in"], w["in_steps"], None, "none", "bf16")
        assert_within(qkv, want, bound)
        for i in range(3):
            rows = slice(count * i, count * (i + 1))
            for n, new in (("k", turned[rows, heads:]), ("v", qkv[rows, (heads + kv_heads) * d:].view(count, kv_heads, d))):
                q, steps = quantised(new)
                held, _ = s.held(n, i, s.lens[i])
                assert torch.equal(held[:, -count:], (q.double() * steps.double()[..., None]).permute(1, 0, 2))
        want, bound = cache_attend_want(s, turned[:, :heads], 1 / math.sqrt(d), "bf16")
        assert_within(o, want, bound)
        want, bound = product_want(*quantised(o.view(s.tokens, -1)), w["out"], w["out_steps"], None, "none", "bf16")
        assert_within(y, want, bound)

    check()
    # captured, and replayed on another input
    first = [t.clone() for t in (qkv, turned, o, y)]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        decoder_step(*args, stream=torch.cuda.current_stream().cuda_stream)
    for t in (qkv, turned, o, y):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, (qkv, turned, o, y)))
    x.copy_(normal(g, s.tokens, width))
    graph.replay()
    torch.cuda.synchronize()
    check()


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 4096, 5000), (1, 47000, 33), (1, 100, 7), (2, 12000, 300), (3, 1003, 257), (4, 11264, 4800), (4, 13000, 100), (2, 17, 1)])
def test_inner_product_of_single_tokens(pkg, element, m, k, n):
    pitch = (k + 15) // 16 * 16
    check_product(pkg, element, m, k, n, "none", w_pitch=pitch)
    check_product(pkg, element, m, k, n, "gelu", x_pitch=k + 3, w_pitch=pitch + 32, w_shift=32)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 3, 40, 300])
def test_weights_written_just_before_a_product(pkg, m):
    """The product's kernels begin early with their weights: what the call before writes has to be there."""
    k, n = 4096, 2048
    g = gen(m)
    x = normal(g, m, k).bfloat16()
    full = [normal(g, n, k) for _ in range(4)]
    w, ws = torch.zeros(n, k, dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda")
    y = [torch.zeros(m, n, device="cuda", dtype=torch.bfloat16) for _ in full]
    space = torch.empty(pkg.op_inner_product_tokens_workspace(m, k), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for f, out in zip(full, y):
        pkg.op_quantize_rows(f.data_ptr(), "f32", n, k, w.data_ptr(), ws.data_ptr())
        pkg.op_inner_product_tokens(x.data_ptr(), out.data_ptr(), "bf16", m, k, n, w.data_ptr(), ws.data_ptr(), space.data_ptr(), space.numel())
    pkg.op_check_status()
    for f, out in zip(full, y):
        want, bound = product_want(*quantised(x), *quantised(f), None, "none", "bf16")
        assert_within(out, want, bound)
