"""How exact the operators of a decoder in 8-bit integers are, whichever kernel a call takes: attention's probabilities."""
import math

import pytest

torch = pytest.importorskip("torch")

from test_decoder_ops import KIND, TINY, U, Setup, assert_within, attend, cache_attend_want, gen, normal  # noqa: E402


def close(s, q, o, element):
    """16-bit types: probabilities in 16 bits (2^-16 of the spread, which is the tolerance of f16 without its own rounding), whatever is
    in the batch; then one rounding to the type."""
    want, bound = cache_attend_want(s, q, 1 / math.sqrt(s.d), "f16")
    return want, bound + U[element] * (want.abs() + bound) + TINY[element]


def run(pkg, s, q, element, shared=0):
    o = torch.zeros_like(q)
    attend(pkg, s, q, o, element, q.shape[1], shared)
    pkg.op_check_status()
    return o


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f16", "bf16"])
@pytest.mark.parametrize("new,lens,heads,kv_heads,d,shared", [
    ([1, 1, 1], [700, 33, 2000], 32, 8, 128, 0), ([150, 40], [900, 333], 8, 2, 128, 0), ([300], [1500], 4, 4, 64, 0), ([1] * 70, [600 + i for i in range(70)], 8, 1, 128, 512),
    ([100, 1], [400, 3000], 16, 4, 72, 0), ([3], [800], 64, 1, 128, 0)])
def test_probabilities_are_held_in_16_bits(pkg, element, new, lens, heads, kv_heads, d, shared):
    s = Setup(pkg, new, lens, kv_heads, d, 16, shared=shared)
    q = normal(gen(3), s.tokens, heads, d).to(KIND[element])
    o = run(pkg, s, q, element, shared)
    assert_within(o, *close(s, q, o, element))


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f16", "bf16"])
@pytest.mark.parametrize("shared", [0, 512])
def test_a_step_is_as_exact_beside_a_prompt_or_behind_a_prefix(pkg, element, shared):
    """The same decoding steps alone and beside a sequence of many new tokens, which takes the batch to the tiles of many rows."""
    lens, heads, kv_heads, d = [900, 700, 2100], 16, 4, 128
    q = normal(gen(5), 103, heads, d).to(KIND[element])
    beside = Setup(pkg, [1, 1, 1, 100], lens + [760], kv_heads, d, 16, shared=shared, seed=7)
    wide = run(pkg, beside, q, element, shared)
    assert_within(wide, *close(beside, q, wide, element))
    # the steps alone, over the same pages
    alone = Setup(pkg, [1, 1, 1], lens, kv_heads, d, 16, seed=7)
    alone.ints, alone.steps, alone.whole, alone.table, alone.pages = beside.ints, beside.steps, beside.whole[:3], beside.table[:3].contiguous(), beside.pages
    alone.table[:, :shared // 16] = alone.table[0, :shared // 16]
    alone.cache = beside.cache
    alone.batch = pkg.CacheBatch(alone.table.data_ptr(), alone.len_t.data_ptr(), alone.starts.data_ptr(), 3, 3, alone.table.shape[1], 1, max(lens))
    few = run(pkg, alone, q[:3].contiguous(), element)
    want, bound = close(alone, q[:3], few, element)
    assert_within(few, want, bound)
    assert_within(wide[:3], want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("count,shared", [(100, 0), (300, 0), (90, 1024)])
def test_maxima_that_rise_with_every_key(pkg, element, d, count, shared):
    """The results so far are scaled down before every half block: behind the products that are under way, each time."""
    s = Setup(pkg, [count] * 3, [1500, 1400, 1300 + count], 2, d, 16, shared=shared)
    s.ints["k"].fill_(100)
    for i, n in enumerate(s.lens):
        keys = torch.arange(n, device="cuda")
        # a score of 10 more with every 64 keys (2^14 in the probability), for the smallest query
        s.steps["k"][s.whole[i].long()[keys // 16], :, keys % 16] = (10 / 64 * keys / (100 * math.sqrt(d)))[:, None]
    q = (1 + normal(gen(6), s.tokens, 8, 1).abs() / 4).expand(-1, -1, d).contiguous().to(KIND[element])
    first = run(pkg, s, q, element, shared)
    assert_within(first, *close(s, q, first, element))
    assert all(torch.equal(first, run(pkg, s, q, element, shared)) for _ in range(20))


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m", [1, 40, 300])
def test_swish_of_numbers_far_below_zero(pkg, element, m):
    """Sums from 0 to -104: the results are numbers of their type down to its smallest one.  A sum of one product is known to the bit, so that
    what is off is the activation alone: fp32's exponential by a step and three roundings (8 F as elsewhere), the fast one by 2 + 1.173 |t|
    steps of 2 F, its quotient by 2; of what is below fp32's smallest normal number a step, twice, times |t|."""
    F, k, n = 2.0 ** -24, 16, 64
    x = torch.zeros(m, k, device="cuda")
    x[:, 0] = 1.0
    w = torch.zeros(n, k, dtype=torch.int8, device="cuda")
    w[:, 0] = -127
    for top in (104.0, 10.0, 1.0):
        ws = torch.linspace(0.0, top / 127, n, device="cuda")
        y = torch.full((m, n), 5.0, device="cuda").to(KIND[element])
        space = torch.empty(pkg.op_inner_product_tokens_workspace(m, k), dtype=torch.uint8, device="cuda")
        pkg.op_inner_product_tokens(x.to(KIND[element]).data_ptr(), y.data_ptr(), element, m, k, n, w.data_ptr(), ws.data_ptr(), space.data_ptr(), space.numel(),
                                    activation="swish")
        torch.cuda.synchronize()
        step = torch.ones(1, device="cuda") / 127
        t = (torch.tensor(-127.0 * 127.0, device="cuda") * (step * ws)).double()
        want = t * torch.sigmoid(t)
        off = want.abs() * 2 * F * (4 if element == "f32" else 5 + 1.2 * t.abs()) + 2 * t.abs() * 2.0 ** -149
        assert_within(y, want.expand(m, n), (off + U[element] * (want.abs() + off) + TINY[element]).expand(m, n))
