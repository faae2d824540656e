"""Group norm, rotary positions and cross attention on device arrays where numbers and calls come to their ends: scores of minus
infinity, shares too small for a type, values far from zero, outliers, errors that belong to somebody else.

Tolerances as in test_device_ops.py: derived from the arithmetic, F = 2^-24, U[t] half a step of type t.
"""
import math

import pytest

torch = pytest.importorskip("torch")

from test_device_ops import KIND, TYPES, U, assert_within, gen, normal


def attend(pkg, q, k, v, element, scale=0.0, lens=None):
    b, lq, heads, d = q.shape
    o = torch.full_like(q, 7.0)
    pkg.op_cross_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), element, b, lq, k.shape[1], heads, k.shape[2], d,
                           None if lens is None else lens.data_ptr(), None, scale)
    torch.cuda.synchronize()
    return o


# ------------------------------------------------------------------------------------------------ cross attention
# queries, keys, heads: a few queries; many over whole blocks of 128 keys, over a last block that is not whole; at most 128 keys
SHAPES = [(1, 512, 2), (200, 512, 80), (100, 640, 80), (200, 500, 80), (700, 128, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("lq,lk,heads", SHAPES)
def test_a_row_whose_scores_are_all_minus_infinity_is_zero(pkg, element, lq, lk, heads):
    """As a row without a key: its sum is 0.  Other rows do not notice."""
    q, k, v = (normal(gen(n), 1, l, heads, 64).to(KIND[element]) for n, l in ((0, lq), (1, lk), (2, lk)))
    k[..., 0] = 1
    want = attend(pkg, q, k, v, element)
    at = lq - 1
    q[0, at, 0] = 0
    q[0, at, 0, 0] = -math.inf
    got = attend(pkg, q, k, v, element)
    assert not got[0, at, 0].any()
    want[0, at, 0] = 0
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk,heads", SHAPES)
def test_shares_below_the_smallest_number_are_zero(pkg, element, lq, lk, heads):
    """Key 0 has all of a row's weight, the others e^-150 = 2^-216 of it each and values of 1e35: they add nothing (1e35 * 2^-216
    * lk is below 1e-27), while a share of 2^-120 would add 0.08 a key.  (Sums of such values stay below fp32's largest.)"""
    q = torch.zeros(1, lq, heads, 64, device="cuda", dtype=KIND[element])
    q[..., 0] = 1
    k = torch.zeros(1, lk, heads, 64, device="cuda", dtype=KIND[element])
    k[:, 1:, :, 0] = -150
    v = torch.full_like(k, 1e35)
    v[:, 0] = 1
    o = attend(pkg, q, k, v, element, 1.0)
    assert torch.equal(o, torch.ones_like(o))
