"""Cache rows appended with the rotation on the way, from graphs that look like the ones fused and are not quite: factors of
another shape, members over memory that died, members in place."""
import numpy as np
import pytest

import latent_ref as ref
from latent_ref import EPS16, EPS32, MROPE, NEOX
from test_latent_gpu import latent_graph, latent_want, positions, rope_node, rope_want, run

pytestmark = pytest.mark.gpu


@pytest.fixture
def ctx(pkg):
    c = pkg.Context()
    yield c
    c.free()


@pytest.mark.parametrize("shape", [(1, 512), (256, 2), (512, 1)])
def test_factors_of_other_shapes(ctx, backend, shape):
    """the norm's factor: one a channel, or as many values that MUL repeats otherwise (one a token of 512 tokens)"""
    rng = np.random.default_rng(shape[0])
    n = 512
    x, w = ctx.new_tensor("f32", 576, n), ctx.new_tensor("f32", *shape)
    pos, kc, ix = ctx.new_tensor("i32", 4 * n), ctx.new_tensor("f32", 576, n), ctx.new_tensor("i64", n)
    row = 4 * 576
    low = ctx.mul(ctx.rms_norm(ctx.view_4d(x, 512, n, 1, 1, row, row * n, row * n, 0), 1e-6), w)
    turned = rope_node(ctx, ctx.view_4d(x, 64, 1, n, 1, row, row, row * n, 2048), pos, MROPE, 64)
    out = ctx.set_rows(kc, ctx.reshape(ctx.concat(ctx.reshape(low, 512, 1, n), turned, 0), 576, n), ix)
    xs, ws = rng.standard_normal((n, 576)).astype(np.float32), (1 + rng.random(shape[::-1])).astype(np.float32)
    p = positions(n, rng)
    got = run(ctx, backend, [out], [(x, xs), (w, ws), (pos, p), (ix, np.arange(n)), (kc, np.zeros((n, 576), np.float32))])[0].reshape(n, 576)
    factor = np.tile(ws.astype(np.float64), (n // shape[1], 512 // shape[0]))
    want = ref.rms_norm(xs[:, :512].astype(np.float64), factor, float(np.float32(1e-6)))
    assert np.all(np.abs(got[:, :512] - want) <= 32 * EPS32 * np.abs(want))


@pytest.mark.parametrize("member", ["norm", "mul", "turned", "norm and turned"])
@pytest.mark.parametrize("mode", [NEOX, MROPE])
def test_members_over_memory_that_died(ctx, backend, member, mode):
    """an allocator that gives a member its input's memory, which nothing reads any more (ggml-alloc's reuse): same rows"""
    rng = np.random.default_rng(1)
    n, n_ctx = 9, 16
    xn, xr, w = ctx.new_tensor("f32", 512, n), ctx.new_tensor("f32", 64, 1, n), ctx.new_tensor("f32", 512)
    pos, kc, ix = ctx.new_tensor("i32", n if mode == NEOX else 4 * n), ctx.new_tensor("f16", 576, n_ctx), ctx.new_tensor("i64", n)
    norm = ctx.rms_norm(xn, 1e-6)
    low = ctx.mul(norm, w)
    turned = rope_node(ctx, xr, pos, mode, 64)
    lowr = ctx.reshape(low, 512, 1, n)
    out = ctx.set_rows(kc, ctx.reshape(ctx.concat(lowr, turned, 0), 576, n), ix)
    twice = ctx.scale(low, 2.0)                                 # (the product is kept: the fused launch writes it as well)
    g = ctx.build(out, twice)
    ctx.alloc(backend)
    if "norm" in member:
        norm.raw.data = xn.raw.data
    if member == "mul":
        low.raw.data = lowr.raw.data = xn.raw.data
    if "turned" in member:
        turned.raw.data = xr.raw.data
    xs, ws = rng.standard_normal((n, 576)).astype(np.float32), (1 + rng.random(512)).astype(np.float32)
    p = np.arange(n, dtype=np.int32) if mode == NEOX else positions(n, rng)
    for t, a in ((xn, xs[:, :512]), (xr, xs[:, 512:]), (w, ws), (pos, p), (ix, np.arange(3, 3 + n)), (kc, np.zeros((n_ctx, 576), np.float16))):
        t.set(a)
    ctx.compute(backend, g)
    want, (tol, mag), kept = latent_want(xs, ws, np.broadcast_to(p, (4, n)), mode, False)
    got = kc.numpy().reshape(n_ctx, 576)
    # one axis: (i + 2) half steps of the angle 8 * 1e4^(-i / 32) from the 32-bit recurrence, under 19 in all
    bound = np.concatenate([tol, (10 + 19) * EPS32 * mag], 1)
    assert np.all(np.abs(got[3:3 + n] - want) <= bound + EPS16 * (np.abs(want) + bound) + 2.0 ** -25) and not got[:3].any() and not got[3 + n:].any()
    assert np.all(np.abs(twice.numpy().reshape(n, 512) - 2 * kept) <= 64 * EPS32 * np.abs(kept))


def test_rotation_in_place(ctx, backend):
    """keys turned in place (ggml_rope_ext_inplace: a view of its input) and appended: the keys themselves turn too"""
    rng = np.random.default_rng(0)
    n, heads, dim = 7, 2, 64
    k, pos, kc, ix = ctx.new_tensor("f32", dim, heads, n), ctx.new_tensor("i32", 4 * n), ctx.new_tensor("f16", dim * heads, 16), ctx.new_tensor("i64", n)
    turned = rope_node(ctx, k, pos, MROPE, dim)
    turned.raw.view_src = k.ptr
    out = ctx.set_rows(kc, ctx.reshape(turned, dim * heads, n), ix)
    ks, p = rng.standard_normal((n, heads, dim)).astype(np.float32), positions(n, rng)
    got = run(ctx, backend, [out], [(k, ks), (pos, p), (ix, np.arange(n)), (kc, np.zeros((16, dim * heads), np.float16))])[0].reshape(16, -1)
    want, mag = rope_want(ks, p, MROPE, dim)
    bound = 10 * EPS32 * mag
    assert np.all(np.abs(k.numpy().reshape(n, heads, dim) - want) <= bound)
    assert np.all(np.abs(got[:n].reshape(n, heads, dim) - want) <= bound + EPS16 * (np.abs(want) + bound) + 2.0 ** -25)
