"""Refusals of the operators for latent attention and several position axes: graph construction needs no GPU."""
import pytest

SEC = (16, 24, 24, 0)


@pytest.fixture
def ctx(pkg):
    c = pkg.Context()
    yield c
    c.free()


def rope_args(ctx, n=5, heads=3, dim=128, type_="f32", pos_n=None, pos_type="i32"):
    return ctx.new_tensor(type_, dim, heads, n), ctx.new_tensor(pos_type, 4 * n if pos_n is None else pos_n)


@pytest.mark.parametrize("mode,n_dims,sections", [(8, 128, SEC), (8, 96, SEC), (40, 128, (24, 20, 20, 0)), (24, 64, (32, 32, 0, 0)), (8, 64, (1, 0, 0, 0))])
def test_rope_multi_accepts(ctx, mode, n_dims, sections):
    x, pos = rope_args(ctx)
    for turn in (ctx.rope_multi, ctx.rope_multi_back):
        y = turn(x, pos, None, n_dims, sections, mode, 8192, 1e6)
        assert y.ne == x.ne and y.op_params(15)[11:15] == list(sections)


@pytest.mark.parametrize("what,kw,call", [
    ("positions of one axis only", dict(pos_n=5), {}),
    ("positions not i32", dict(pos_type="f32"), {}),
    ("odd n_dims", {}, dict(n_dims=127)),
    ("more n_dims than channels", {}, dict(n_dims=256)),
    ("no channel turns", {}, dict(n_dims=0)),
    ("vision with n_dims not half", {}, dict(mode=24)),
    ("a mode of one axis", {}, dict(mode=2)),
    ("an unknown mode", {}, dict(mode=12)),
    ("empty sections", {}, dict(sections=(0, 0, 0, 0))),
    ("a negative section", {}, dict(sections=(64, -1, 1, 0))),
    ("integers", dict(type_="i32"), {}),
    ("more pairs than the table holds", dict(dim=2048), dict(n_dims=2048)),
])
def test_rope_multi_refuses(ctx, what, kw, call):
    x, pos = rope_args(ctx, **kw)
    a = dict(n_dims=128, sections=SEC, mode=8)
    a.update(call)
    for turn in (ctx.rope_multi, ctx.rope_multi_back):
        with pytest.raises(RuntimeError):
            turn(x, pos, None, a["n_dims"], a["sections"], a["mode"], 8192, 1e6)


def test_rope_refuses_short_frequency_factors(ctx):
    x, pos = rope_args(ctx)
    with pytest.raises(RuntimeError):
        ctx.rope_multi(x, pos, ctx.new_tensor("f32", 63), 128, SEC, 8, 8192, 1e6)
    with pytest.raises(RuntimeError):
        ctx.rope_ext_back(x, ctx.new_tensor("i32", 4), None, 128, 2, 8192, 1e6)


def test_concat_refuses(ctx):
    a = ctx.new_tensor("f32", 8, 3, 2)
    for b, dim in [(ctx.new_tensor("f16", 8, 3, 2), 0), (ctx.new_tensor("f32", 8, 4, 2), 0), (a, 4), (a, -1)]:
        with pytest.raises(RuntimeError):
            ctx.concat(a, b, dim)
    with pytest.raises(RuntimeError):
        ctx.concat(ctx.new_tensor("q8_0", 32, 2), ctx.new_tensor("q8_0", 32, 2), 1)
    assert ctx.concat(a, ctx.new_tensor("f32", 8, 5, 2), 1).ne == (8, 8, 2, 1)


def wide(ctx, cache="f16", dk=576, dv=512, tok=2, heads=4, n_kv=9, kv_heads=1, seqs=1, kv_seqs=None, off=0, q_type="f32", mask=None, shared=True):
    q = ctx.new_tensor(q_type, dk, tok, heads, seqs)
    k = ctx.new_tensor(cache, dk, n_kv, kv_heads, kv_seqs or seqs)
    nb = k.nb
    v = ctx.view_4d(k, dv, n_kv, kv_heads, kv_seqs or seqs, nb[1], nb[2], nb[3], off) if shared else ctx.new_tensor(cache, dv, n_kv, kv_heads, kv_seqs or seqs)
    return ctx.flash_attn_ext(q, k, v, mask(ctx) if mask else None, 0.07)


@pytest.mark.parametrize("kw", [
    {}, dict(cache="q8_0"), dict(cache="q4_0"), dict(off=128), dict(cache="q8_0", off=68), dict(heads=7), dict(seqs=3), dict(seqs=3, kv_seqs=1),
    dict(dk=192, dv=128, kv_heads=4, shared=False), dict(dk=192, dv=128, kv_heads=2, shared=False), dict(kv_heads=2),
    dict(mask=lambda c: c.new_tensor("f16", 9, 2)), dict(mask=lambda c: c.new_tensor("f16", 16, 64)), dict(mask=lambda c: c.new_tensor("f16", 9, 2, 4)),
])
def test_wide_attention_accepts(ctx, kw):
    assert wide(ctx, **kw).ne == (kw.get("dv", 512), kw.get("heads", 4), 2, kw.get("seqs", 1))


@pytest.mark.parametrize("what,kw", [
    ("values of their own", dict(shared=False)),
    ("values elsewhere in the row", dict(off=64)),
    ("a width that has no kernel", dict(dk=320, dv=256)),
    ("q in half precision", dict(q_type="f16")),
    ("a cache type without a kernel", dict(cache="q4_1")),
    ("a bf16 cache", dict(cache="bf16")),
    ("expanded keys in 8 bits", dict(dk=192, dv=128, kv_heads=4, shared=False, cache="q8_0")),
    ("heads that the KV heads do not divide", dict(kv_heads=3)),
    ("fewer KV streams than sequences", dict(seqs=4, kv_seqs=2)),
    ("a mask of fewer keys", dict(mask=lambda c: c.new_tensor("f16", 8, 2))),
    ("a mask of fewer tokens", dict(mask=lambda c: c.new_tensor("f16", 9, 1))),
    ("a mask in 32 bits", dict(mask=lambda c: c.new_tensor("f32", 9, 2))),
    ("a mask whose heads do not divide", dict(mask=lambda c: c.new_tensor("f16", 9, 2, 3))),
    ("no keys", dict(n_kv=0)),
])
def test_wide_attention_refuses(ctx, what, kw):
    with pytest.raises(RuntimeError):
        wide(ctx, **kw)


def test_equal_widths_unchanged(ctx):
    q, k, v = ctx.new_tensor("f32", 128, 2, 4), ctx.new_tensor("f16", 128, 9, 2), ctx.new_tensor("f16", 128, 9, 2)
    assert ctx.flash_attn_ext(q, k, v, None, 0.1).ne == (128, 4, 2, 1)
