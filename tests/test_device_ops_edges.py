"""Group norm, rotary positions and cross attention on device arrays where numbers and calls come to their ends: scores of minus
infinity, shares too small for a type, values far from zero, outliers, errors that belong to somebody else.

Tolerances as in test_device_ops.py: derived from the arithmetic, F = 2^-24, U[t] half a step of type t.
"""
import math
import threading

import pytest

torch = pytest.importorskip("torch")

from test_device_ops import F, KIND, TYPES, U, assert_within, attend_want, check_attend, check_norm, check_rotary, gen, normal, rotary_want


def attend(pkg, q, k, v, element, scale=0.0, lens=None):
    b, lq, heads, d = q.shape
    o = torch.full_like(q, 7.0)
    pkg.op_cross_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), element, b, lq, k.shape[1], heads, k.shape[2], d,
                           None if lens is None else lens.data_ptr(), None, scale)
    torch.cuda.synchronize()
    return o


# ------------------------------------------------------------------------------------------------ whose error it is
@pytest.mark.gpu
@pytest.mark.parametrize("earlier", ["no such device", "no room"])
def test_an_earlier_error_is_not_this_call_s(pkg, tmp_path, earlier):
    """A load that asks for a device that is not there, and a batch that no device has room for, fail; operators afterwards run."""
    param, bin_ = pkg.zoo.single_conv(str(tmp_path / "conv"))
    x = normal(gen(1), 2, 64, 4, 64)
    positions = torch.zeros(128, 1, device="cuda", dtype=torch.int32)
    calls = [lambda y: pkg.op_group_norm(x.data_ptr(), y.data_ptr(), "f32", 2, 64, 256, 8),
             lambda y: pkg.op_rotary_axes(x.data_ptr(), y.data_ptr(), "f32", 128, 4, 64, positions.data_ptr(), [32]),
             lambda y: pkg.op_cross_attention(x.data_ptr(), x.data_ptr(), x.data_ptr(), y.data_ptr(), "f32", 2, 64, 64, 4, 4, 64),
             lambda y: pkg.op_cross_attention(x.data_ptr(), x.data_ptr(), x.data_ptr(), y.data_ptr(), "bf16", 1, 64, 64, 4, 4, 64),
             lambda y: pkg.op_cross_attention(x.data_ptr(), x.data_ptr(), x.data_ptr(), y.data_ptr(), "bf16", 2, 1, 64, 4, 4, 64)]
    model = pkg.Model(param, bin_)
    for call in calls:
        if earlier == "no room":
            assert model.launch_count(1 << 20) < 0
        else:
            with pytest.raises(pkg.NcnnB200Error):
                pkg.Model(param, bin_, device=99)
        call(torch.empty_like(x))
    torch.cuda.synchronize()


def stalled_call(pkg, device="cuda"):
    """A call whose first block of keys never arrives: its waits run out after 2 ms."""
    q, k, v = (torch.randn(1, l, 2, 64, device=device).half() for l in (200, 300, 300))
    o = torch.empty_like(q)
    L = pkg.load_library()
    L.ncnn_b200_op_test_hooks(1, 2000000, 0)
    try:
        pkg.op_cross_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), "f16", 1, 200, 300, 2, 2, 64)
    finally:
        L.ncnn_b200_op_test_hooks(0, 0, 0)
    torch.cuda.synchronize(device)


def status(pkg):
    try:
        pkg.op_check_status()
    except pkg.NcnnB200Error as e:
        return e.status
    return 0


@pytest.mark.gpu
def test_every_thread_is_told_of_a_wait_that_ran_out(pkg):
    """A thread that asks first takes the answer from no other; each gets it once."""
    status(pkg)
    stalled_call(pkg)
    others = []
    t = threading.Thread(target=lambda: others.extend([status(pkg), status(pkg)]))
    t.start()
    t.join()
    assert others == [7, 0]
    assert [status(pkg), status(pkg)] == [7, 0]
    stalled_call(pkg)
    assert [status(pkg), status(pkg)] == [7, 0]


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_a_wait_that_ran_out_on_another_device_is_told(pkg):
    status(pkg)
    stalled_call(pkg, "cuda:1")
    assert torch.cuda.current_device() == 0
    assert [status(pkg), status(pkg)] == [7, 0]


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


@pytest.mark.gpu
def test_the_environment_of_the_host_is_not_read_by_a_call(pkg, monkeypatch):
    """Another thread may be changing it.  The Python binding passes NCNN_B200_TEST_STALL on through ncnn_b200_op_test_hooks."""
    q, k, v = (normal(gen(n), 1, l, 2, 64).half() for n, l in ((0, 200), (1, 300), (2, 300)))
    o = torch.empty_like(q)
    pkg.op_check_status()
    monkeypatch.setenv("NCNN_B200_TEST_STALL", "1")
    L = pkg.load_library()
    assert L.ncnn_b200_op_cross_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), 1, 1, 200, 300, 2, 2, 64, None, None, None, 0.0, None) == 0
    monkeypatch.delenv("NCNN_B200_TEST_STALL")
    pkg.op_check_status()
    assert torch.isfinite(o).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk,heads", [(200, 300, 2), (100, 300, 80), (700, 100, 64)])
def test_a_kernel_of_other_registers_is_refused_by_its_name(pkg, lq, lk, heads):
    """setmaxnreg would wait without a limit there.  The message speaks of registers, nothing is launched, later calls are right."""
    q, k, v = (normal(gen(n), 1, l, heads, 64).half() for n, l in ((0, lq), (1, lk), (2, lk)))
    want = attend(pkg, q, k, v, "f16")
    o = torch.full_like(q, 5.0)
    L = pkg.load_library()
    L.ncnn_b200_op_test_hooks(0, 0, 24)
    try:
        with pytest.raises(pkg.NcnnB200Error, match="registers") as err:
            pkg.op_cross_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), "f16", 1, lq, lk, heads, heads, 64)
    finally:
        L.ncnn_b200_op_test_hooks(0, 0, 0)
    assert err.value.status == 6
    torch.cuda.synchronize()
    assert (o == 5.0).all()
    assert torch.equal(attend(pkg, q, k, v, "f16"), want)


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [100, 200])
def test_a_walk_over_the_keys_may_take_longer_than_a_wait(pkg, lq):
    """2^20 keys take some 10 ms, each step a microsecond; the limit of a wait is 2 ms here.  The sequence ends before the array and
    inside a step of 16 keys: one warp waits for the last block from the start."""
    lk, heads = 1 << 20, 80
    q, k, v = (normal(gen(n), 1, l, h, 64).to(torch.bfloat16) for n, l, h in ((0, lq, heads), (1, lk, 1), (2, lk, 1)))
    lens = torch.tensor([lk - 3], device="cuda", dtype=torch.int32)
    status(pkg)
    want = attend(pkg, q, k, v, "bf16", lens=lens)
    L = pkg.load_library()
    L.ncnn_b200_op_test_hooks(0, 2000000, 0)
    try:
        got = attend(pkg, q, k, v, "bf16", lens=lens)
    finally:
        L.ncnn_b200_op_test_hooks(0, 0, 0)
    assert status(pkg) == 0
    assert torch.isfinite(got).all() and torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("element", ["f16", "bf16"])
@pytest.mark.parametrize("lq,lk,heads,sinks", [(130, 131072, 80, 1), (1, 1 << 22, 1, 128)])
def test_many_keys_of_little_weight_behind_few_of_much(pkg, element, lq, lk, heads, sinks):
    """Key 0 (or the first keys of 128 tiles of 16, one to each warp of the cluster that shares out a query's keys) at a score of 0 and
    value 0, all others at -17.375 (2^-25.07) and value 1: the result is their share.  Scores are exact.  Sums: up to lk / 16 steps of
    the products, which truncate (2 F each), and lk / 64 additions of a thread.  An fp16 probability is off by 2^-32 of a sink at
    most, a bf16 one by its rounding; the result's own rounding."""
    q = torch.zeros(1, lq, heads, 64, device="cuda", dtype=KIND[element])
    q[..., 0] = 1
    k = torch.zeros(1, lk, 1, 64, device="cuda", dtype=KIND[element])
    k[..., 0] = -17.375
    v = torch.ones_like(k)
    k[0, 0:16 * sinks:16, 0, 0] = 0
    v[0, 0:16 * sinks:16] = 0
    o = attend(pkg, q, k, v, element, 1.0)
    weak = (lk - sinks) * math.exp(-17.375)
    want = torch.full_like(o, weak / (weak + sinks), dtype=torch.float64)
    off = (lk / 16 * 2 + lk / 64) * F + 2.0 ** -20 + U[element]
    lost = 2.0 ** -32 * lk / sinks if element == "f16" else U[element] * want
    assert_within(o, want, off * want + lost)


def test_a_scale_past_the_largest_number_is_refused(pkg):
    """The kernels multiply scores by scale / ln 2; infinite, it would make a NaN of a score of 0."""
    import numpy as np

    keep = [np.zeros(64, np.float32) for _ in range(4)]
    q, k, v, o = (a.ctypes.data for a in keep)
    for scale, says in ((2.4e38, "scale"), (3.4e38, "scale"), (2.3e38, "device memory"), (1e-45, "device memory")):
        with pytest.raises(pkg.NcnnB200Error, match=says) as err:
            pkg.op_cross_attention(q, k, v, o, "f32", 1, 1, 1, 1, 1, 8, scale=scale)
        assert err.value.status == 2


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("lq,lk,heads,kv_heads", [(1, 3000, 8, 2), (20, 5000, 2, 1), (150, 700, 4, 4), (600, 100, 40, 40)])
def test_a_sequence_alone_has_its_value_of_a_batch(pkg, element, lq, lk, heads, kv_heads):
    """Keys may be cut over other CTAs than in a batch: the same value within the arithmetic's bound, not always the same bits."""
    q, k, v = (normal(gen(n), 3, l, h, 64).to(KIND[element]) for n, l, h in ((0, lq, heads), (1, lk, kv_heads), (2, lk, kv_heads)))
    batch, alone = attend(pkg, q, k, v, element), attend(pkg, q[1:2], k[1:2], v[1:2], element)
    want, bound = attend_want(q[1:2], k[1:2], v[1:2], torch.ones(1, lk, dtype=torch.bool, device="cuda"), 0.125, element)
    assert_within(alone, want, bound)
    assert_within(batch[1:2], want, bound)


# ------------------------------------------------------------------------------------------------ group norm
@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("in_place", [False, True])
def test_groups_wider_than_a_cta(pkg, element, in_place):
    """Groups of more than 256 accesses of channels (16-byte ones, or what the address and the channels allow), one and several of
    them, whole tensors and ranges of a wider one's channels; at most 2^9 values to a thread, as norm_want counts."""
    wide = 2056 if element != "f32" else 1028
    check_norm(pkg, element, 1, 60, wide, 1, "none", in_place=in_place)
    check_norm(pkg, element, 3, 41, 2 * wide, 2, "swish", in_place=in_place)
    check_norm(pkg, element, 2, 1, wide, 1, "relu", in_place=in_place)
    check_norm(pkg, element, 2, 7, 5140, 1, "gelu", affine=False, in_place=in_place)
    check_norm(pkg, element, 2, 130, 300, 1, "gelu", shift=1, in_place=in_place)
    check_norm(pkg, element, 1, 90, 771, 3, "swish", x_pitch=773, y_pitch=773 if in_place else 771, in_place=in_place)


def check_statistics(pkg, x, groups, terms):
    """Against the formula in 64 bits; `terms`: the values of a thread.  A thread's sums of differences from a shift near the mean
    are off by `terms` F of the sum of their sizes (two deviations a value at most), its squares' likewise; its first 64 may stand
    about an outlier, whose square their sums then lose 64 * 64 / 2 F of.  Joining 256 threads and 16 CTAs adds 2^8 F of six
    deviations and the mean's own rounding, 3 F of its size."""
    n, p, c = x.shape
    y = torch.empty_like(x)
    pkg.op_group_norm(x.data_ptr(), y.data_ptr(), "f32", n, p, c, groups, None, None, 1e-5, "none")
    t = x.double().view(n, p, groups, c // groups)
    mean = t.mean((1, 3), keepdim=True)
    sd = torch.sqrt((t - mean).square().mean((1, 3), keepdim=True) + 1e-5)
    z = (t - mean) / sd
    dm = (2 * terms + 6 * 2.0 ** 8) * F + 3 * F * mean.abs() / sd
    assert_within(y, z.reshape(n, p, c), (dm + z.abs() * ((terms + 2.0 ** 11) * F + dm * dm + 8 * F)).reshape(n, p, c))


@pytest.mark.gpu
@pytest.mark.parametrize("pixels,mean", [(16384, 1003.0), (65536, 1003.0), (4096, 0.0)])
def test_groups_wider_than_a_cta_far_from_zero(pkg, pixels, mean):
    """Sums of so many values about zero would put the mean off by 0.2 (16384 pixels) and 2 deviations (65536)."""
    x = normal(gen(1), 1, pixels, 1028) + mean
    check_statistics(pkg, x, 1, pixels * 1028 // 256)


@pytest.mark.gpu
@pytest.mark.parametrize("outlier", [1e3, 1e5])
def test_groups_wider_than_a_cta_with_an_outlier(pkg, outlier):
    """The first value of a thread far from all others."""
    x = normal(gen(1), 1, 4096, 1028)
    x[0, 0, 0] = outlier
    check_statistics(pkg, x, 1, 4096 * 1028 // 256)


@pytest.mark.gpu
def test_groups_wider_than_a_cta_constant_and_nonfinite(pkg):
    """A group of one value is beta; a NaN or an infinity stays in its own group of its own image."""
    x = torch.full((2, 37, 2060), 3.0, device="cuda")
    x[1] = normal(gen(1), 37, 2060)
    x[1, 5, 2] = math.nan
    y = torch.empty_like(x)
    beta = torch.arange(2060, device="cuda", dtype=torch.float32)
    pkg.op_group_norm(x.data_ptr(), y.data_ptr(), "f32", 2, 37, 2060, 2, None, beta.data_ptr(), 1e-5, "relu")
    assert torch.equal(y[0], beta.expand(37, 2060))
    assert torch.isnan(y[1, :, :1030]).all() and torch.isfinite(y[1, :, 1030:]).all()
    x[1, 5, 2] = math.inf
    pkg.op_group_norm(x.data_ptr(), y.data_ptr(), "f32", 2, 37, 2060, 2, None, beta.data_ptr(), 1e-5, "relu")
    assert torch.isnan(y[1, 5, 2]) and torch.isfinite(y[1, :, 1030:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("outlier", [1e2, 1e3, 1e4, 1e5])
@pytest.mark.parametrize("pixels,channels,terms", [(65536, 255, 4096), (262144, 32, 512)])
def test_group_norm_with_an_outlier(pkg, outlier, pixels, channels, terms):
    """The first value of a thread far from all others (16 CTAs to the group, one or 32 rows of threads)."""
    x = normal(gen(1), 1, pixels, channels)
    x[0, 0, 0] = outlier
    check_statistics(pkg, x, 1, terms)


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [64, 1028])
def test_swish_of_fp32_is_good_to_fp32(pkg, channels):
    """Against the formula on the values without an activation, which are the same.  2^t is off by 4 F of itself (the instruction's
    2^-22), its correction, 1 + e, the reciprocal after a Newton step and the product by F each, the reciprocal's remainder by less
    than F: 9 F.  (An argument rounded once would add F for every unit of it.)  Above -80 nothing leaves fp32's range."""
    x = normal(gen(1), 1, 2000, channels)
    gamma = torch.full((channels,), 15.0, device="cuda")
    line, got = torch.empty_like(x), torch.empty_like(x)
    for y, act in ((line, "none"), (got, "swish")):
        pkg.op_group_norm(x.data_ptr(), y.data_ptr(), "f32", 1, 2000, channels, 1, gamma.data_ptr(), None, 1e-5, act)
    line = line.double()
    assert -80 < line.min() < -50
    want = line * torch.sigmoid(line)
    assert_within(got, want, 9 * F * want.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
def test_swish_at_the_ends_of_the_numbers(pkg, element):
    """A gamma of 0 leaves beta: far negative values give 0, far positive ones themselves, minus infinity and NaN a NaN."""
    values = [math.inf, 3e38, 1e30, 200.0, 100.0, 88.5, 0.0, -0.0, -88.5, -100.0, -200.0, -1e30, -3e38, -math.inf, math.nan, 1.0]
    x = normal(gen(1), 1, 50, 16).to(KIND[element])
    y = torch.empty_like(x)
    gamma, beta = torch.zeros(16, device="cuda"), torch.tensor(values, device="cuda")
    pkg.op_group_norm(x.data_ptr(), y.data_ptr(), element, 1, 50, 16, 4, gamma.data_ptr(), beta.data_ptr(), 1e-5, "swish")
    got = y[0].float()
    assert torch.equal(got[:, :13], got[:1, :13].expand(50, 13))
    assert torch.equal(y[0, 0, :6], beta[:6].to(KIND[element]))
    assert (got[:, 6:13].abs() < 1e-35).all()
    assert torch.isnan(got[:, 13:15]).all()


# ------------------------------------------------------------------------------------------------ rotary positions
ONE_OF = [(1, 4, (0, 64, 0, 64)), (1, 4, (64, 64, 8, 80)), (1, 4, (7, 65, 3, 66)), (5, 1, (64, 0, 64, 0)), (5, 1, (80, 8, 72, 3)), (1, 1, (0, 0, 0, 0)),
          (1, 4, (0, 0, 0, 64))]


@pytest.mark.parametrize("tokens,heads,strides", ONE_OF)
def test_the_stride_of_an_axis_of_one_entry_says_nothing(pkg, tokens, heads, strides):
    """One token's, or one head's, step is never taken: host memory is what is refused here, not strides."""
    import numpy as np

    keep = [np.zeros(1024, np.float32) for _ in range(3)]
    x, y, positions = (a.ctypes.data for a in keep)
    with pytest.raises(pkg.NcnnB200Error, match="device memory"):
        pkg.op_rotary_axes(x, y, "f32", tokens, heads, 64, positions, [32], strides=strides)
    with pytest.raises(pkg.NcnnB200Error, match="device memory"):  # in place: strides that are stepped with have to agree
        pkg.op_rotary_axes(x, x, "f32", tokens, heads, 64, positions, [32],
                           strides=(strides[2] + (8 if tokens == 1 else 0), strides[3] + (8 if heads == 1 else 0), *strides[2:]))


def test_strides_that_are_stepped_with_are_still_refused(pkg):
    import numpy as np

    keep = [np.zeros(1024, np.float32) for _ in range(3)]
    x, y, positions = (a.ctypes.data for a in keep)
    for tokens, heads, strides in ((1, 4, (0, 64, 0, 63)), (5, 1, (64, 0, 63, 0)), (2, 2, (128, 64, 64, 64)), (1, 4, (-1, 64, 0, 64)), (5, 1, (64, 0, 64, -1)),
                                   (2, 2, (128, 64, 100, 64))):
        with pytest.raises(pkg.NcnnB200Error, match="strides"):
            pkg.op_rotary_axes(x, y, "f32", tokens, heads, 64, positions, [32], strides=strides)
    for tokens, heads, strides in ((2, 1, (64, 64, 72, 64)), (1, 2, (64, 64, 64, 72))):
        with pytest.raises(pkg.NcnnB200Error, match="in place"):
            pkg.op_rotary_axes(x, x, "f32", tokens, heads, 64, positions, [32], strides=strides)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_of_one_token_or_one_head(pkg, element, interleaved):
    for tokens, heads, strides in ONE_OF[:-1]:
        check_rotary(pkg, element, tokens, heads, 64, [10, 16], interleaved, False, strides=strides)
    check_rotary(pkg, element, 1, 4, 64, [10, 16], interleaved, True, strides=(0, 64, 0, 64), in_place=True)


def test_a_negative_number_of_positions_is_refused(pkg):
    """0 stands for one to each token; below that is a mistake of the caller, whose array may have any size."""
    import numpy as np

    keep = [np.zeros(1024, np.float32) for _ in range(3)]
    x, y, positions = (a.ctypes.data for a in keep)
    for rows, says in ((-1, "position_rows"), (-(1 << 40), "position_rows"), (0, "device memory"), (2, "device memory"), (1 << 40, "device memory")):
        with pytest.raises(pkg.NcnnB200Error, match=says) as err:
            pkg.op_rotary_axes(x, y, "f32", 2, 1, 64, positions, [32], position_rows=rows)
        assert err.value.status == 2


@pytest.mark.gpu
@pytest.mark.parametrize("base", [1.01, 2.0, 10000.0])
def test_angles_of_far_positions_of_slow_spectra(pkg, base):
    """Frequencies close to one another and positions at the ends of their type, against 60 digits: 2^-25 of a turn, sincospif's own
    2 F, and F for each product with (1, 0)."""
    from decimal import Decimal, getcontext

    getcontext().prec = 60
    turn = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    at = [0, 1, -1, (1 << 31) - 1, -(1 << 31), 2000000011, -1999999973, 123456789]
    positions = torch.tensor(at, dtype=torch.int32, device="cuda").view(-1, 1).contiguous()
    x = torch.zeros(len(at), 1, 256, device="cuda")
    x[..., :128] = 1
    y = torch.empty_like(x)
    pkg.op_rotary_axes(x.data_ptr(), y.data_ptr(), "f32", len(at), 1, 256, positions.data_ptr(), [128], base)
    want = torch.empty(len(at), 256, dtype=torch.float64)
    for i, p in enumerate(at):
        for j in range(128):
            part = p * (-Decimal(base).ln() * j / 128).exp() / turn
            angle = 2 * math.pi * float(part - part.to_integral_value())
            want[i, j], want[i, 128 + j] = math.cos(angle), math.sin(angle)
    assert_within(y.view(len(at), 256), want.cuda(), torch.full((len(at), 256), 2 * math.pi * 2.0 ** -25 + 4 * F, device="cuda"))


# ------------------------------------------------------------------------------------------------ the ends of the ranges
@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
def test_more_images_than_a_grid_has_rows(pkg, element):
    check_norm(pkg, element, 70000, 3, 4, 2, "swish")
    check_norm(pkg, element, 66000, 2, 6, 2, "none", in_place=True, x_pitch=7, y_pitch=7)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
def test_the_most_sequences_and_heads(pkg, element):
    q, k, v = (normal(gen(n), 65535, l, 1, 8).to(KIND[element]) for n, l in ((0, 1), (1, 3), (2, 3)))
    o = attend(pkg, q, k, v, element)
    p = torch.softmax((q.double() * k.double()).sum(-1)[:, :, 0] * 8 ** -0.5, 1)
    want, spread = (p[..., None] * v[:, :, 0].double()).sum(1), (p[..., None] * v[:, :, 0].double().abs()).sum(1)
    # attend_want's bound for 8 components and 3 keys of sizes up to 6: scores to 24 F * 6 * 6 * 8 / sqrt(8), the probability's rounding
    rel = 2 * 24 * F * 6 * 6 * 8 ** 0.5 + 28 * F + (U[element] if element != "f32" else 0)
    assert_within(o[:, 0, 0], want, rel * spread + U[element] * (want.abs() + rel * spread) + 2.0 ** -23 * v.abs().max() * (element == "f16") + 2.0 ** -25)
    q = normal(gen(0), 1, 1, 65535, 8).to(KIND[element])
    k, v = (normal(gen(n), 1, 40, 1, 8).to(KIND[element]) for n in (1, 2))
    o = attend(pkg, q, k, v, element)
    # every head reads the same keys: heads are queries of one head
    want, bound = attend_want(q.view(1, 65535, 1, 8), k, v, torch.ones(1, 40, dtype=torch.bool, device="cuda"), 8 ** -0.5, element)
    assert_within(o.view(1, 65535, 1, 8), want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("element", TYPES)
@pytest.mark.parametrize("lq", [1, 140])
def test_keys_and_values_that_overlap_in_memory(pkg, element, lq):
    """Windows of one signal: rows of 64 components, 8 (and 4) elements from one to the next."""
    for step in (8, 4):
        check_attend(pkg, element, 1, lq, 300, 2, 1, 64, strides=(lq * 128, 128, 64, 0, step, 64, 0, step, 64, lq * 128, 128, 64))


@pytest.mark.gpu
def test_rotary_of_more_threads_than_a_launch(pkg):
    """2^23 + 70 tokens of 128 pairs at an odd address, 2^30 pairs to a launch: the last tokens belong to a second one, and positions
    repeat through both."""
    tokens, rows, d = (1 << 23) + 70, 1000, 256
    x = torch.empty(tokens * d + 1, device="cuda", dtype=torch.float16)
    view = x[1:].view(tokens, d)
    some = torch.cat([torch.arange(0, 40), torch.arange((1 << 23) - 40, tokens)]).cuda()
    view.zero_()
    view[some] = normal(gen(1), some.numel(), d).half()
    positions = torch.randint(-1000, 1000, (rows, 2), generator=gen(2), device="cuda", dtype=torch.int64).to(torch.int32)
    want, mag = rotary_want(view[some].view(-1, 1, d), positions[some % rows], [64, 64], 10000.0, True, False)
    pkg.op_rotary_axes(x.data_ptr() + 2, x.data_ptr() + 2, "f16", tokens, 1, d, positions.data_ptr(), [64, 64], 10000.0, True, False, rows)
    assert_within(view[some].view(-1, 1, d), want, 10 * F * mag + U["f16"] * (want.abs() + 10 * F * mag) + 2.0 ** -25)
    assert not view[1 << 20].any()
