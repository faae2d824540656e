"""The kernels that large calls of a decoder's operators take.  Which one a size takes goes by the device's SMs: each test says which one it
is for and asks the same rule, so that a size that has come to another kernel fails."""
import time

import pytest

torch = pytest.importorskip("torch")

from test_decoder_ops import (KIND, Setup, assert_within, attend, cache_attend_want, check_product, check_rows, gen, normal, product_want,  # noqa: E402
                              quantised, strided)


def up(a, b):
    return (a + b - 1) // b


def product_kernel(m, k, n):
    """("one",), ("few", tokens of a tile, CTAs that share its K blocks, CTAs of the call) or ("pair", channels of a tile)."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    if m <= 2 and m * up(k, 512) * 512 <= 46 * 1024:
        return ("one",)
    if up(m, 128) * up(n, 128) <= 2 * sms:
        columns = 128 if m >= 128 else up(m, 16) * 16
        while m > 64 and columns > 32 and 2 * up(m, columns) * up(n, 128) <= sms:
            columns = up(columns // 2, 16) * 16
        tiles, ranks = up(m, columns) * up(n, 128), 1
        while ranks < 8 and tiles * ranks * 2 <= sms and ranks * 2 <= up(k, 128):
            ranks *= 2
        return ("few", columns, ranks, tiles * ranks)
    busiest = {c: up(up(m, 256) * up(n, c), sms // 2) * c for c in (128, 256)}
    return ("pair", 128 if busiest[128] < busiest[256] else 256)


def status(pkg):
    try:
        pkg.op_check_status()
        return 0
    except pkg.NcnnB200Error as e:
        return e.status


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f32", "bf16"])
@pytest.mark.parametrize("kernel,m,k,n", [(("few", 128, 1), 200, 256, 12000), (("few", 16, 8), 16, 2048, 256), (("few", 128, 1), 1024, 1040, 4096),
                                          (("pair", 128), 2100, 144, 4100), (("pair", 256), 3000, 1040, 3000)])
def test_a_wait_that_runs_out_in_each_kernel(pkg, monkeypatch, element, kernel, m, k, n):
    """Of a pair of CTAs, one has copies in flight then, the other has none.  Waits end after 2 ms here, and those for the copies when
    these have landed, not when 0.2 s are over."""
    assert product_kernel(m, k, n)[:len(kernel)] == kernel
    assert status(pkg) == 0
    x, w, ws = normal(gen(1), m, k).to(KIND[element]), torch.ones(n, k, dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda")
    y, space = torch.zeros(m, n, device="cuda").to(x.dtype), torch.empty(pkg.op_inner_product_tokens_workspace(m, k), dtype=torch.uint8, device="cuda")
    monkeypatch.setenv("NCNN_B200_TEST_STALL", "1")
    pkg.op_inner_product_tokens(x.data_ptr(), y.data_ptr(), element, m, k, n, w.data_ptr(), ws.data_ptr(), space.data_ptr(), space.numel())
    began = time.perf_counter()
    torch.cuda.synchronize()
    assert time.perf_counter() - began < 0.15
    assert status(pkg) == 7 and status(pkg) == 0
    monkeypatch.delenv("NCNN_B200_TEST_STALL")
    check_product(pkg, element, m, k, n)
    assert status(pkg) == 0


def check(pkg, element, m, k, n, act="none", bias=True, y_pitch=0, shift=0, aligned=True):
    """A product against the formula: results `shift` elements into their array, steps and bias at multiples of 16 bytes or not."""
    g = gen(m + k + n)
    yp, size = y_pitch or n, KIND[element].itemsize
    x = normal(g, m, k).to(KIND[element])
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    y = torch.full((m * yp + shift,), 5.0, device="cuda", dtype=KIND[element])
    at = 0 if aligned else 1
    ws = ((normal(g, n + 1).abs() + 0.2) / (40 * k ** 0.5))[at:at + n]
    b = normal(g, n + 1)[at:at + n] if bias else None
    space = torch.empty(pkg.op_inner_product_tokens_workspace(m, k), dtype=torch.uint8, device="cuda")
    pkg.op_inner_product_tokens(x.data_ptr(), y.data_ptr() + shift * size, element, m, k, n, w.data_ptr(), ws.data_ptr(), space.data_ptr(), space.numel(),
                                None if b is None else b.data_ptr(), act, y_pitch=yp)
    assert status(pkg) == 0
    q, steps = quantised(x)
    want, bound = product_want(q, steps, w, ws, b, act, element)
    assert_within(torch.as_strided(y, (m, n), (yp, 1), shift), want, bound)
    if yp > n:
        assert bool((torch.as_strided(y, (m - 1, yp - n), (yp, 1), shift + n) == 5.0).all())
    assert bool((y[:shift] == 5.0).all())


SIZES = [(("pair", 128), 2100, 144, 4100), (("pair", 128), 2048, 2064, 3000), (("pair", 256), 3000, 272, 3000), (("pair", 256), 3000, 1040, 2960),
         (("few", 128, 1), 1024, 272, 4096), (("few", 128, 1), 1000, 1040, 4000)]


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "relu", "swish", "gelu"])
@pytest.mark.parametrize("kernel,m,k,n", SIZES)
def test_large_products(pkg, element, act, kernel, m, k, n):
    took = product_kernel(m, k, n)
    assert took[:len(kernel)] == kernel and (kernel[0] == "pair" or took[3] > torch.cuda.get_device_properties(0).multi_processor_count)  # (two CTAs to an SM)
    check(pkg, element, m, k, n, act, bias=act != "none")


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kernel,m,k,n", SIZES)
def test_large_products_in_other_layouts(pkg, element, kernel, m, k, n):
    assert product_kernel(m, k, n)[:len(kernel)] == kernel
    check(pkg, element, m, k, n, "swish", y_pitch=n + 1)                       # (no row but the first where TMA could store it)
    check(pkg, element, m, k, n, "gelu", y_pitch=n + (-n) % 8 + 24)            # (TMA stores into the pitch's rows, not between them)
    check(pkg, element, m, k, n, "none", shift=1)
    check(pkg, element, m, k, n, "relu", aligned=False)
    check(pkg, element, m, k, n, "none", y_pitch=n + 3, shift=3, aligned=False)


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,m,k,n", SIZES)
def test_large_products_of_tokens_that_are_no_numbers(pkg, kernel, m, k, n):
    x = normal(gen(m), m, k).bfloat16()
    bad = [0, 127, 128, 255, 256, m - 1]
    x[bad, 3] = float("inf")
    w, ws = torch.randint(-127, 128, (n, k), generator=gen(1), device="cuda", dtype=torch.int8), torch.full((n,), 1e-3, device="cuda")
    y, space = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16), torch.empty(pkg.op_inner_product_tokens_workspace(m, k), dtype=torch.uint8, device="cuda")
    for act in ("none", "relu", "swish", "gelu"):
        pkg.op_inner_product_tokens(x.data_ptr(), y.data_ptr(), "bf16", m, k, n, w.data_ptr(), ws.data_ptr(), space.data_ptr(), space.numel(), activation=act)
        assert status(pkg) == 0
        rows = torch.isnan(y)
        assert bool(rows[bad].all()) and int(rows.any(1).sum()) == len(bad)


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,columns", [(2048, 8), (2049, 4096), (5000, 1000), (3001, 2048), (2050, 4104), (2048, 520)])
def test_many_rows_to_integers(pkg, element, rows, columns):
    """From 2048 rows on a warp takes a row that it can keep (4096 columns, 2048 of f32)."""
    g = gen(rows + columns)
    x = (normal(g, rows, columns) * normal(g, columns).abs()).to(KIND[element])
    x[5], x[rows - 1, 0], x[rows - 2, columns - 1], x[7, 0] = 0.0, float("nan"), float("-inf"), torch.finfo(KIND[element]).max
    check_rows(pkg, x, element)
    check_rows(pkg, x, element, columns + 24, 8)


def places(s):
    """Row, page (-1: none) and row of the page of every token, as tensors."""
    rows, pages, at = [], [], []
    for i, count in enumerate(s.new):
        j = torch.arange(count, device="cuda")
        position = s.lens[i] - count + j
        page = s.whole[i].long()[(position // s.page).clamp_min(0)]
        rows.append(s.firsts[i] + j)
        pages.append(torch.where((position >= 0) & (page >= 0) & (page < s.pages), page, -1))
        at.append(position % s.page)
    return torch.cat(rows), torch.cat(pages), torch.cat(at)


def check_many_rows(pkg, element, s, strides=None, shift=0):
    g = gen(1)
    kind, size = KIND[element], KIND[element].itemsize
    four = None if strides is None else (*strides, *strides)
    rows, pages, at = places(s)
    there = pages >= 0
    src = {n: strided(g, kind, s.tokens, s.kv_heads, s.d, strides, shift) for n in "kv"}
    want = {n: (s.ints[n].clone(), s.steps[n].clone()) for n in "kv"}
    for n in "kv":
        q, steps = quantised(src[n][1][rows[there]])
        want[n][0][pages[there], :, at[there]] = torch.nn.functional.pad(q, (0, s.row - s.d))
        want[n][1][pages[there], :, at[there]] = steps
    pkg.op_cache_write(s.cache, s.batch, src["k"][0].data_ptr() + shift * size, src["v"][0].data_ptr() + shift * size, element, four)
    torch.cuda.synchronize()
    for n in "kv":
        assert torch.equal(s.ints[n], want[n][0]) and torch.equal(torch.nan_to_num(s.steps[n], nan=-1.0), torch.nan_to_num(want[n][1], nan=-1.0))
    for names in ("kv", "k", "v"):
        out = {n: strided(g, kind, s.tokens, s.kv_heads, s.d, strides, shift) for n in names}
        for n in names:
            view = torch.as_strided(want_out := out[n][0].clone(), out[n][1].shape, out[n][1].stride(), shift)
            view[rows] = torch.where(there[:, None, None], (s.ints[n][pages, :, at, :s.d].float() * s.steps[n][pages, :, at][..., None]).to(kind), 0.0)
            out[n] = (*out[n], want_out)
        pkg.op_cache_read(s.cache, s.batch, *((out[n][0].data_ptr() + shift * size if n in out else None) for n in "kv"), element, four)
        torch.cuda.synchronize()
        for n in names:
            assert torch.equal(out[n][0], out[n][2])


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv_heads,d,page,strides,shift", [(8, 128, 64, None, 0), (3, 72, 16, None, 0), (6, 64, 32, (400, 64), 8), (5, 200, 16, None, 0), (7, 33, 16, None, 1),
                                                          (2, 128, 128, (300, 137), 3), (6, 40, 16, (40, 40 * 30000), 0)])
def test_many_rows_of_a_cache(pkg, element, kv_heads, d, page, strides, shift):
    """Four heads to a lane, where keys or values alone fill the device: the ends of heads, tokens, pages and pieces of rows."""
    row = (d + 15) // 16 * 16
    most = 4096 * torch.cuda.get_device_properties(0).multi_processor_count
    tokens = up(most, kv_heads * row // 8) + 77
    new = [tokens // 2, 0, 1, tokens // 3, tokens - tokens // 2 - tokens // 3 - 1]
    lens = [new[0] + 1000, 5, 40, new[3] - 20, new[4] + 3]  # (one has more rows than tokens: the first 20 have no place)
    s = Setup(pkg, new, lens, kv_heads, d, page, behind=5, lead=3, fill=False)
    assert tokens * kv_heads * (row // 8) >= most
    for bad in (-1, s.pages, 1 << 30):
        page_of = (1000 + new[0] // 2) // page
        s.whole[0, page_of] = s.table[0, page_of] = bad
        s.whole[3, 0] = s.table[3, 0] = bad
        check_many_rows(pkg, element, s, strides, shift)


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kernel,m,n", [(("pair", 128), 2100, 4100), (("pair", 256), 3000, 3000), (("few", 128, 1), 1024, 4096)])
def test_large_products_of_rows_that_end_inside_16_bytes(pkg, element, kernel, m, n):
    """Anything may lie behind a row of weights, and in the workspace behind a token's integers."""
    for k, pitch in ((100, 112), (1, 16), (129, 176)):
        assert product_kernel(m, k, n)[:2] == kernel[:2]
        check_product(pkg, element, m, k, n, "none", w_pitch=pitch, x_pitch=k + 3)


@pytest.mark.gpu
@pytest.mark.parametrize("n,y_pitch", [(16384, 16400), (16399, 16400)])
def test_results_past_32_bits(pkg, n, y_pitch):
    """More than 2^32 results, through TMA and without it."""
    m, k = 270000, 48
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("not enough device memory")
    g = gen(2)
    x = normal(g, m, k).bfloat16()
    w, ws = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8), normal(g, n).abs()
    y = torch.full((m, y_pitch), 5.0, device="cuda", dtype=torch.bfloat16)
    space = torch.empty(pkg.op_inner_product_tokens_workspace(m, k), dtype=torch.uint8, device="cuda")
    pkg.op_inner_product_tokens(x.data_ptr(), y.data_ptr(), "bf16", m, k, n, w.data_ptr(), ws.data_ptr(), space.data_ptr(), space.numel(), y_pitch=y_pitch)
    assert status(pkg) == 0
    for rows in (slice(0, 300), slice(261000, 263000), slice(m - 700, m)):
        want, bound = product_want(*quantised(x[rows]), w, ws, None, "none", "bf16")
        assert_within(y[rows, :n], want, bound)
        assert bool((y[rows, n:] == 5.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f32", "bf16"])
@pytest.mark.parametrize("heads,shared", [(4, 0), (4, 64), (64, 0), (64, 64)])
def test_one_row_to_a_sequence_and_more_rows_or_sequences_than_the_other(pkg, element, heads, shared):
    """Without starts, row s is sequence s's: sequences behind the last row have none, rows behind the last sequence are left alone."""
    kv_heads, d, lens = 1, 64, [90, 70, 200, 65, 333]
    for rows, sequences in ((3, 5), (5, 3), (9, 5)):
        s = Setup(pkg, [1] * 5, lens, kv_heads, d, 16, shared=shared, starts=False)
        s.batch = pkg.CacheBatch(s.table.data_ptr(), s.len_t.data_ptr(), None, sequences, rows, s.width, 0, 0)
        used = min(rows, sequences)
        q = normal(gen(1), rows, heads, d).to(KIND[element])
        o = torch.full_like(q, 5.0)
        attend(pkg, s, q, o, element, heads, shared)
        assert status(pkg) == 0
        s.new, s.lens, s.firsts = [1] * used, lens[:used], list(range(used + 1))
        want, bound = cache_attend_want(s, q[:used], d ** -0.5, element)
        assert_within(o[:used], want, bound)
        assert bool((o[used:] == 5.0).all())
        k = normal(gen(2), rows, kv_heads, d).to(KIND[element])
        back = torch.full_like(k, 5.0)
        before = {n: s.ints[n].clone() for n in "kv"}
        pkg.op_cache_write(s.cache, s.batch, k.data_ptr(), k.data_ptr(), element)
        pkg.op_cache_read(s.cache, s.batch, back.data_ptr(), None, element)
        torch.cuda.synchronize()
        integers, steps = quantised(k[:used])
        assert torch.equal(back[:used], (integers.float() * steps[..., None]).to(KIND[element])) and bool((back[used:] == 5.0).all())
        for n in "kv":
            page = [int(s.whole[i, (lens[i] - 1) // 16]) for i in range(used)]
            for i in range(used):
                before[n][page[i], :, (lens[i] - 1) % 16, :d] = integers[i]
            assert torch.equal(s.ints[n][..., :d], before[n][..., :d])
