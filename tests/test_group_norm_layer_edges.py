"""GroupNorm layers of loaded graphs beside other readers of their operand, and groups that a graph does not take."""
import numpy as np
import pytest

from conftest import rel_l2
from test_group_norm_layer import TOL, graph, refusal

F = 2.0 ** -24


def test_groups_that_no_cta_holds_are_refused_at_load(pkg, tmp_path):
    """256 threads of four channels each (of one, where the channels are no multiple of four), over whole accesses."""
    for channels, groups in ((1028, 1), (257, 1), (2056, 2), (514, 2), (1028, 4)):  # (the last: only all four groups are whole accesses)
        status, message = refusal(pkg, tmp_path, f"0={groups} 1={channels}", f"0=2 1=2 2={channels}", (np.ones(channels), np.zeros(channels)))
        assert status == 8 and "so many channels" in message, (channels, groups)
    for channels, groups in ((1024, 1), (255, 1), (2048, 2), (510, 2), (1024, 4)):
        weights = (np.ones(channels), np.zeros(channels))
        param, bin_ = graph(pkg, tmp_path / "m", [("Input", "input", [], ["data"], f"0=2 1=2 2={channels}"),
                                                  ("GroupNorm", "norm", ["data"], ["output"], f"0={groups} 1={channels}")], weights)
        assert pkg.Model(param, bin_, plan_only=True).output_shapes == [(channels, 2, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("first", ["", "ReLU"])
@pytest.mark.parametrize("c,groups", [(64, 8), (36, 4)])
def test_an_operand_that_a_convolution_reads_too(pkg, oracle, tmp_path, mode, first, c, groups):
    """A map of mean 1000 deviations, normalised and convolved: the group norm reads all of its 24 bits, whatever format the
    convolution wants (a bf16 pair would leave steps of 2^-6 to 2^-7 of a deviation, tf32 half a deviation)."""
    h, w = 16, 12
    net = pkg.zoo._Net(5)
    wr = net.w
    wr.layer("Input", "input", [], ["data"], f"0={w} 1={h} 2={c}")
    if first:
        wr.layer(first, "first", ["data"], ["map"], "")
    wr.layer("Split", "split", ["map" if first else "data"], ["a", "b", "d"])
    net.conv("conv1", "b", "c1", c, 32, 1, 1, 0, act=0, zero_bias=False)
    wr.layer("GroupNorm", "norm", ["a"], ["n"], f"0={groups} 1={c} 2=1e-5 3=0")
    net.conv("conv3", "d", "c3", c, 32, 3, 1, 1, act=0, zero_bias=False)
    param, bin_ = wr.save(str(tmp_path / "m"))
    x = (np.random.default_rng(3).standard_normal((3, c, h, w)) + 1000).astype(np.float32)
    model = pkg.Model(param, bin_, accuracy_mode=mode)
    got = dict(zip(model.output_names, model.run(x)))
    t = x.astype(np.float64).reshape(3, groups, -1)
    mean, sd = t.mean(-1, keepdims=True), np.sqrt(t.var(-1, keepdims=True) + 1e-5)
    want = ((t - mean) / sd).reshape(x.shape)
    # a thread's sums of at most 2^9 differences and their joining: 2^10 F of a deviation; the mean's own rounding: 3 F of its size;
    # the variance: 2^11 F of itself
    bound = 2.0 ** 10 * F + 3 * F * (np.abs(mean) / sd).max() + np.abs(want) * (2.0 ** 11 + 8) * F
    assert (np.abs(got["n"] - want) <= bound).all()
    reference = oracle.Model(param, bin_)
    for i, xi in enumerate(x):
        for name, value in zip(model.output_names, reference.run([xi])):
            if name != "n":
                assert rel_l2(got[name][i], value) < TOL[mode]
    # a batch is its images run alone, bit for bit, and the same without a captured graph
    plain = pkg.Model(param, bin_, accuracy_mode=mode, use_cuda_graph=False)
    for name, alone, value in zip(model.output_names, model.run(x[2]), plain.run(x)):
        assert np.array_equal(got[name][2], alone) and np.array_equal(got[name], value)


@pytest.mark.gpu
def test_a_batch_that_is_uploaded_in_pieces(pkg, tmp_path, monkeypatch):
    """16 MB of inputs: the first layers run piece by piece while the next piece is on its way, with the bits of the whole batch."""
    param, bin_ = pkg.zoo.group_norm_block(str(tmp_path / "block"), h=64, w=64, c=64, cout=32, groups=8)
    x = (np.random.default_rng(1).standard_normal((16, 64, 64, 64)) + 3).astype(np.float32)
    got = pkg.Model(param, bin_).run(x)[0]
    monkeypatch.setenv("NCNN_B200_PIPELINE", "0")
    assert np.array_equal(got, pkg.Model(param, bin_).run(x)[0])
