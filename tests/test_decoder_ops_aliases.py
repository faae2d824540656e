"""Arrays of the operators of a decoder in 8-bit integers that start at one address where one of them is written: refused (no GPU)."""
import pytest

torch = pytest.importorskip("torch")

from test_decoder_ops import batch_of, cache_of, host  # noqa: E402


def refused(pkg, call):
    with pytest.raises(pkg.NcnnB200Error, match="must not lie over|memory of their own") as err:
        call()
    return err.value.status == 2


def test_products_whose_arrays_are_one(pkg):
    keep = [host() for _ in range(6)]
    x, y, w, ws, bias, space = (k[1] for k in keep)

    def call(**change):
        a = {**dict(x=x, y=y, w=w, ws=ws, bias=bias, space=space), **change}
        return lambda: pkg.op_inner_product_tokens(a["x"], a["y"], "f32", 2, 4, 3, a["w"], a["ws"], a["space"], 1 << 20, a["bias"])

    for written in ("y", "space"):
        for other, at in dict(x=x, w=w, ws=ws, bias=bias, y=y, space=space).items():
            if other != written:
                assert refused(pkg, call(**{written: at})), (written, other)
    with pytest.raises(pkg.NcnnB200Error, match="device memory"):
        call()()


def test_cache_calls_whose_arrays_are_one(pkg):
    keep = [host() for _ in range(10)]
    at = [k[1] for k in keep]
    starts = at[9]
    cache, batch = cache_of(pkg, at), batch_of(pkg, at[4:], starts=starts)
    a, b, space = at[6:9]
    # (k, v, k_steps, v_steps, table, lens, starts)
    for other in at[:6] + [starts]:
        assert refused(pkg, lambda: pkg.op_cache_write(cache, batch, a, other, "f32"))
        assert refused(pkg, lambda: pkg.op_cache_read(cache, batch, other, b, "f32"))
        assert refused(pkg, lambda: pkg.op_cache_attention(cache, batch, a, other, "f32", 4, workspace_ptr=space, workspace_bytes=1 << 20))
        assert refused(pkg, lambda: pkg.op_cache_attention(cache, batch, a, b, "f32", 4, workspace_ptr=other, workspace_bytes=1 << 20))
    for q, o, room in ((a, a, space), (a, b, a), (a, b, b)):
        assert refused(pkg, lambda: pkg.op_cache_attention(cache, batch, q, o, "f32", 4, workspace_ptr=room, workspace_bytes=1 << 20))
    for change in (dict(k_steps=at[0]), dict(v_steps=at[0]), dict(k_steps=at[1]), dict(v_steps=at[1])):
        assert refused(pkg, lambda: pkg.op_cache_write(cache_of(pkg, at, **change), batch, a, b, "f32"))
    with pytest.raises(pkg.NcnnB200Error, match="device memory"):
        pkg.op_cache_attention(cache, batch, a, b, "f32", 4, workspace_ptr=space, workspace_bytes=1 << 20)
