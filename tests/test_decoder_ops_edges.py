"""The operators of a decoder in 8-bit integers where they meet one another, the device's limits and calls that nobody makes on purpose."""
import math
import threading

import pytest

torch = pytest.importorskip("torch")

from test_decoder_ops import (Setup, attend, assert_within, cache_attend_want, check_attention, check_product, check_write_read, gen, normal,  # noqa: E402
                              product_want, quantised, status_of)


def status(pkg):
    try:
        pkg.op_check_status()
        return 0
    except pkg.NcnnB200Error as e:
        return e.status


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["few", "few ranks", "pair", "cache", "cache f16", "cache prefix"])
def test_a_wait_that_runs_out_is_reported(pkg, monkeypatch, what):
    assert status(pkg) == 0
    monkeypatch.setenv("NCNN_B200_TEST_STALL", "1")
    if what.startswith("cache"):
        kind = torch.float16 if what == "cache f16" else torch.bfloat16
        shared = 64 if what == "cache prefix" else 0
        s = Setup(pkg, [40] * 3, [300, 200, 104], 2, 64, 16, shared=shared)
        q = normal(gen(1), s.tokens, 4, 64).to(kind)
        o = torch.zeros_like(q)
        element = "f16" if what == "cache f16" else "bf16"
        space = attend(pkg, s, q, o, element, 4, shared)
    else:
        m, k, n = {"few": (200, 256, 20000), "few ranks": (16, 2048, 256), "pair": (2048, 256, 3000)}[what]
        x, w, ws = normal(gen(1), m, k), torch.ones(n, k, dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda")
        y, space = torch.zeros(m, n, device="cuda"), torch.empty(pkg.op_inner_product_tokens_workspace(m, k), dtype=torch.uint8, device="cuda")
        pkg.op_inner_product_tokens(x.data_ptr(), y.data_ptr(), "f32", m, k, n, w.data_ptr(), ws.data_ptr(), space.data_ptr(), space.numel())
    assert status(pkg) == 7
    assert status(pkg) == 0
    monkeypatch.delenv("NCNN_B200_TEST_STALL")
    # the device is as it was, and so are the operators
    if what.startswith("cache"):
        check_attention(pkg, element, s, 4, shared)
    else:
        check_product(pkg, "f32", m, k, n)
    assert status(pkg) == 0


@pytest.mark.gpu
def test_a_kernel_of_other_registers_is_refused(pkg):
    s = Setup(pkg, [100], [300], 2, 128, 16)
    q = normal(gen(1), s.tokens, 8, 128).bfloat16()
    o = torch.full_like(q, 7.0)
    L = pkg.load_library()
    L.ncnn_b200_op_test_hooks(0, 0, 40)
    try:
        assert status_of(lambda: attend(pkg, s, q, o, "bf16", 8)) == 6
    finally:
        L.ncnn_b200_op_test_hooks(0, 0, 0)
    torch.cuda.synchronize()
    assert bool((o == 7.0).all())
    check_attention(pkg, "bf16", s, 8)


@pytest.mark.gpu
def test_calls_at_once(pkg):
    """Calls of several threads on streams of their own, each with its own workspace, give what they give alone."""
    cases = []
    for i, (count, lens, shared, element) in enumerate([(1, [900, 40, 333], 0, "f16"), (70, [700, 90, 300], 0, "bf16"), (1, [600, 700, 520], 512, "bf16"), (3, [100, 50, 9], 0, "f32")]):
        s = Setup(pkg, [count] * 3, [max(n, count) for n in lens], 2, 128, 16, shared=shared, seed=i)
        q = normal(gen(i), s.tokens, 8, 128).to({"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[element])
        want = torch.zeros_like(q)
        attend(pkg, s, q, want, element, 8, shared)
        pkg.op_check_status()
        cases.append((s, q, want, element, shared))
    g = gen(9)
    k, n = 1024, 640
    w, ws = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8), normal(g, n).abs()
    products = []
    for m in (1, 17, 300):
        x = normal(g, m, k).bfloat16()
        y = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
        space = torch.empty(pkg.op_inner_product_tokens_workspace(m, k), dtype=torch.uint8, device="cuda")
        pkg.op_inner_product_tokens(x.data_ptr(), y.data_ptr(), "bf16", m, k, n, w.data_ptr(), ws.data_ptr(), space.data_ptr(), space.numel())
        pkg.op_check_status()
        products.append((m, x, y))
    errors = []

    def attends(case):
        s, q, want, element, shared = case
        stream = torch.cuda.Stream()
        space = torch.empty(max(16, pkg.op_cache_attention_workspace(s.cache, s.batch, 8, shared)), dtype=torch.uint8, device="cuda")
        o = torch.zeros_like(q)
        torch.cuda.synchronize()
        for _ in range(20):
            attend(pkg, s, q, o, element, 8, shared, stream=stream.cuda_stream, space=space)
        stream.synchronize()
        if not torch.equal(o, want):
            errors.append(element)

    def multiplies(case):
        m, x, want = case
        stream = torch.cuda.Stream()
        space = torch.empty(pkg.op_inner_product_tokens_workspace(m, k), dtype=torch.uint8, device="cuda")
        y = torch.zeros_like(want)
        torch.cuda.synchronize()
        for _ in range(20):
            pkg.op_inner_product_tokens(x.data_ptr(), y.data_ptr(), "bf16", m, k, n, w.data_ptr(), ws.data_ptr(), space.data_ptr(), space.numel(), stream=stream.cuda_stream)
        stream.synchronize()
        if not torch.equal(y, want):
            errors.append(m)

    threads = [threading.Thread(target=attends, args=(c,)) for c in cases] + [threading.Thread(target=multiplies, args=(c,)) for c in products]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and status(pkg) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("count,shared", [(1, 0), (1, 256), (60, 0), (60, 256)])
def test_two_graphs_that_share_a_workspace(pkg, count, shared):
    """Replayed one after the other on a stream, and with lengths that changed between replays."""
    s = Setup(pkg, [count] * 4, [400 + count, 300 + count, 270 + count, 256 + count], 2, 128, 16, shared=shared)
    qs = [normal(gen(i), s.tokens, 8, 128).bfloat16() for i in range(2)]
    outs = [torch.zeros_like(q) for q in qs]
    space = attend(pkg, s, qs[0], outs[0], "bf16", 8, shared)
    torch.cuda.synchronize()
    graphs = []
    for q, o in zip(qs, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attend(pkg, s, q, o, "bf16", 8, shared, stream=torch.cuda.current_stream().cuda_stream, space=space)
        graphs.append(graph)
    for step in range(3):
        for graph in graphs:
            graph.replay()
        pkg.op_check_status()
        for q, o in zip(qs, outs):
            want, bound = cache_attend_want(s, q, 1 / math.sqrt(128), "bf16")
            assert_within(o, want, bound)
        s.lens = [n - 40 for n in s.lens] if step == 0 else [n + 17 for n in s.lens]  # (the longest are those of the call)
        s.len_t.copy_(torch.tensor(s.lens, dtype=torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f32", "bf16"])
def test_starts_and_lengths_of_any_value_stay_inside(pkg, element):
    """Arrays that break their rules: nothing outside the call's arrays is read or written."""
    kind = torch.float32 if element == "f32" else torch.bfloat16
    for count in (2, 50):
        s = Setup(pkg, [count] * 3, [count + 90, count + 20, count], 2, 64, 16)
        tokens = s.tokens
        guard = 64
        for starts, lens in (([0, 1 << 30, -5, tokens], s.lens), ([-7, -3, tokens + 100, 3], s.lens), ([tokens, 0, tokens, 0], [1 << 30, -1, -(1 << 31)]),
                             ([0, count, 2 * count, 3 * count], [(1 << 31) - 1] * 3)):
            s.starts.copy_(torch.tensor(starts, dtype=torch.int32))
            s.len_t.copy_(torch.tensor(lens, dtype=torch.int32))
            q = normal(gen(1), tokens, 4, 64).to(kind)
            buf = torch.full((tokens + 2 * guard, 4, 64), 3.0, device="cuda", dtype=kind)
            attend(pkg, s, q, buf[guard:], element, 4)
            x = normal(gen(2), tokens, 2, 64).to(kind)
            pkg.op_cache_write(s.cache, s.batch, x.data_ptr(), x.data_ptr(), element)
            back = torch.full((tokens + 2 * guard, 2, 64), 3.0, device="cuda", dtype=kind)
            pkg.op_cache_read(s.cache, s.batch, back[guard:].data_ptr(), None, element)
            assert status(pkg) == 0
            for t in (buf, back):
                assert bool((t[:guard] == 3.0).all()) and bool((t[tokens + guard:] == 3.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
def test_many_sequences_and_heads(pkg, element):
    s = Setup(pkg, [1] * 700, [1 + i % 37 for i in range(700)], 1, 32, 16, starts=False)
    check_attention(pkg, element, s, 3)
    s = Setup(pkg, [1] * 3, [20, 1, 33], 300, 16, 16, starts=False)
    check_attention(pkg, element, s, 300)
    check_write_read(pkg, element, Setup(pkg, [1] * 3, [20, 1, 33], 300, 16, 16, fill=False, starts=False))
    s = Setup(pkg, [2, 1], [70, 9], 1, 128, 16)
    check_attention(pkg, element, s, 64)  # (128 rows to a key head)


@pytest.mark.gpu
def test_a_prefix_longer_than_any_sequence(pkg):
    for count, element in ((1, "f32"), (1, "bf16"), (40, "bf16")):
        s = Setup(pkg, [count] * 3, [100, 64, max(count, 3)], 2, 64, 16, shared=96)
        # the table's first row reaches 112: more than the sequences' own tokens lie in the prefix
        check_attention(pkg, element, s, 4, shared=96)


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
def test_relu_and_swish_of_large_sums(pkg, element):
    """Activations far out: no NaN from an exponential that overflows, ReLU of a sum below any number."""
    m, k, n = 5, 64, 48
    x = torch.ones(m, k, device="cuda").to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[element])
    w = torch.full((n, k), -127, dtype=torch.int8, device="cuda")
    w[::2] = 127
    ws = torch.logspace(-6, 1.5, n, device="cuda")
    space = torch.empty(pkg.op_inner_product_tokens_workspace(m, k), dtype=torch.uint8, device="cuda")
    for act in ("relu", "swish", "gelu"):
        y = torch.zeros(m, n, device="cuda", dtype=x.dtype)
        pkg.op_inner_product_tokens(x.data_ptr(), y.data_ptr(), element, m, k, n, w.data_ptr(), ws.data_ptr(), space.data_ptr(), space.numel(), activation=act)
        torch.cuda.synchronize()
        want, bound = product_want(*quantised(x), w, ws, None, act, element)
        fits = want.abs() < torch.finfo(x.dtype).max
        assert_within(torch.where(fits, y.double(), 0.0), torch.where(fits, want, 0.0), bound)
