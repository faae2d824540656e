"""The kernels that large calls of a decoder's operators take.  Which one a size takes goes by the device's SMs: each test says which one it
is for and asks the same rule, so that a size that has come to another kernel fails."""
import time

import pytest

torch = pytest.importorskip("torch")

from test_decoder_ops import KIND, assert_within, check_product, gen, normal, product_want, quantised  # noqa: E402


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
