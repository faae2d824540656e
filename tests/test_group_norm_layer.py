"""GroupNorm as a layer of a loaded graph (ncnn's parameters: 0=group 1=channels 2=eps 3=affine), with the activation behind it
fused, against the oracle."""
import numpy as np
import pytest

from conftest import rel_l2

TOL = {0: 1e-4, 1: 5e-3, 2: 4e-6}  # as the other networks of two convolutions, by accuracy mode; normalising adds 2e-6


def graph(pkg, prefix, layers, weights=()):
    w = pkg.zoo._Writer()
    for layer in layers:
        w.layer(*layer)
    for a in weights:
        w.f32(a)
    return w.save(str(prefix))


def refusal(pkg, tmp_path, params, shape="0=4 1=4 2=8", weights=(np.ones(8), np.zeros(8))):
    param, bin_ = graph(pkg, tmp_path / "m", [("Input", "input", [], ["data"], shape), ("GroupNorm", "norm", ["data"], ["output"], params)], weights)
    with pytest.raises(pkg.NcnnB200Error) as err:
        pkg.Model(param, bin_, plan_only=True)
    return err.value.status, str(err.value)


def test_refusals_and_shapes(pkg, tmp_path):
    for params, shape in (("0=3 1=8", "0=4 1=4 2=8"), ("0=0 1=8", "0=4 1=4 2=8"), ("0=-2 1=8", "0=4 1=4 2=8"), ("0=2 1=0", "0=4 1=4 2=8"),
                          ("0=2 1=8 3=2", "0=4 1=4 2=8"), ("0=2 1=8 2=-1e-3", "0=4 1=4 2=8"), ("0=2 1=8", "0=4 1=4 2=6"), ("0=2 1=8", "0=8 1=4"), ("0=2 1=8", "0=8")):
        status, message = refusal(pkg, tmp_path, params, shape)
        assert status == 8 and message, (params, shape)
    assert refusal(pkg, tmp_path, "0=2 1=8", weights=(np.ones(8),))[0] == 8  # a .bin that ends early
    param, bin_ = pkg.zoo.group_norm_block(str(tmp_path / "block"), h=5, w=7, c=32, cout=48, groups=8)
    m = pkg.Model(param, bin_, plan_only=True)
    assert m.output_shapes == [(48, 5, 7)]


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("h,w,c,cout,groups,act,affine,n", [(16, 16, 64, 96, 32, "Swish", True, 3), (9, 13, 32, 40, 8, "GELU", True, 2), (7, 5, 12, 20, 4, "ReLU", False, 1),
                                                            (40, 36, 64, 64, 1, "Swish", True, 2), (3, 3, 24, 24, 24, "Sigmoid", True, 5), (33, 31, 6, 9, 3, "Swish", True, 2)])
def test_block_of_an_image_generator(pkg, oracle, tmp_path, mode, h, w, c, cout, groups, act, affine, n):
    param, bin_ = pkg.zoo.group_norm_block(str(tmp_path / "block"), h=h, w=w, c=c, cout=cout, groups=groups, act=act, affine=affine)
    x = (np.random.default_rng(h).standard_normal((n, c, h, w)) * 2 + 0.7).astype(np.float32)
    reference = oracle.Model(param, bin_)
    want = np.stack([reference.run([xi])[0] for xi in x])
    model = pkg.Model(param, bin_, accuracy_mode=mode)
    got = model.run(x)[0]
    assert rel_l2(got, want) < TOL[mode]
    # a batch is its images run alone, bit for bit, and the same without a captured graph
    assert np.array_equal(got[n - 1], model.run(x[n - 1])[0])
    assert np.array_equal(got, pkg.Model(param, bin_, accuracy_mode=mode, use_cuda_graph=False).run(x)[0])
    kernels = [row["kernel"] for row in model.profile(n, 1)]
    fused = act in ("Swish", "GELU", "ReLU")
    assert kernels.count("k_group_norm") == 2 and kernels.count("k_unary") == (0 if fused else 2)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((1, 1, 1), 1), ((64, 1, 1), 8), ((5, 9, 11), 5), ((256, 30, 30), 32), ((1000, 3, 2), 1)])
def test_layer_alone(pkg, oracle, tmp_path, shape, groups):
    """Graph input to graph output; ncnn's default eps of 0.001."""
    c, h, w = shape
    rng = np.random.default_rng(c)
    param, bin_ = graph(pkg, tmp_path / "m", [("Input", "input", [], ["data"], f"0={w} 1={h} 2={c}"), ("GroupNorm", "norm", ["data"], ["output"], f"0={groups} 1={c}")],
                        (rng.standard_normal(c), rng.standard_normal(c)))
    x = (rng.standard_normal((3, c, h, w)) + 3).astype(np.float32)
    reference = oracle.Model(param, bin_)
    want = np.stack([reference.run([xi])[0] for xi in x])
    got = pkg.Model(param, bin_).run(x)[0]
    # fp32 statistics: off by some 2^-20 of values of the size of one, offsets of one
    assert np.abs(got - want).max() <= 2.0 ** -16 * (1 + np.abs(want).max())
