"""The kernels that large calls of a decoder's operators take.  Which one a size takes goes by the device's SMs: each test says which one it
is for and asks the same rule, so that a size that has come to another kernel fails."""
import time

import pytest

torch = pytest.importorskip("torch")

from test_decoder_ops import KIND, Setup, assert_within, check_product, check_rows, gen, normal, product_want, quantised, strided  # noqa: E402


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
