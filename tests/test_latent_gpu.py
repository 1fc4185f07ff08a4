"""Rotary positions with several axes and their gradient, rotated cache rows, CONCAT, and attention whose keys are
wider than its values (latent attention), against 64-bit references (latent_ref.py).

Bounds. ROPE: the angle is reduced in 64 bits, so cos and sin are off by the rounding of the reduced turn (pi 2^-24)
and sincospi's (2 ulp, 2^-23), then the scale, two products and a sum: under 10 * 2^-24 of |a| + |b| for an output of
the pair (a, b); an f16 result adds 2^-11 of itself. NORM: a sum of n squares in f32 and a square root, under
(n^0.5 / 2 + 8) 2^-24 with n / 256 serial terms a thread: 32 * 2^-24 of the value. Attention: with 22-bit terms and f32
sums a score of O(1) is off by about 3e-7 (18 steps of 2^-24, random), its weight by as much of itself, the result by
the same of its norm: 2e-6 of the norm is six times that, and a seventieth of what one rounding of q to 11 bits costs.
"""
import ctypes

import numpy as np
import pytest

import latent_ref as ref
from latent_ref import EPS16, EPS32, EPSBF, IMROPE, MROPE, NEOX, NORMAL, VISION, rel

pytestmark = pytest.mark.gpu

ATT_REL = 2e-6
SECTIONS = {MROPE: (16, 24, 24, 0), IMROPE: (24, 20, 20, 0), VISION: (32, 32, 0, 0), NORMAL: None, NEOX: None}


@pytest.fixture
def ctx(pkg):
    c = pkg.Context()
    yield c
    c.free()


def run(ctx, backend, outs, feeds, times=1):
    g = ctx.build(*outs)
    ctx.alloc(backend)
    for t, a in feeds:
        t.set(a)
    for _ in range(times):
        ctx.compute(backend, g)
    return [o.numpy() for o in outs]


def positions(n, rng, far=30000):
    p = np.sort(rng.integers(0, far, (4, n)), axis=1).astype(np.int32)
    p[:, 0] = far
    return p


# ---- ROPE with several axes, ROPE_BACK ---------------------------------------------------------------
ROPE_CASES = [  # mode, n, heads, dim, n_dims, sections
    (MROPE, 1, 32, 128, 128, (16, 24, 24, 0)), (MROPE, 7, 3, 128, 128, (16, 24, 24, 0)), (MROPE, 5, 2, 128, 96, (16, 24, 8, 0)),
    (MROPE, 1500, 1, 64, 64, (8, 12, 12, 0)), (MROPE, 3, 5, 12, 12, (2, 2, 1, 1)), (MROPE, 2, 2, 128, 128, (3, 4, 5, 2)),
    (IMROPE, 9, 4, 128, 128, (24, 20, 20, 0)), (IMROPE, 4, 2, 96, 96, (18, 15, 15, 0)), (IMROPE, 3, 2, 128, 128, (11, 11, 10, 0)),
    (VISION, 49, 16, 80, 40, (20, 20, 0, 0)), (VISION, 6, 3, 64, 32, (16, 16, 0, 0)), (VISION, 4, 1, 128, 64, (16, 16, 16, 16)),
    (MROPE, 2, 1, 1024, 1024, (200, 156, 156, 0)), (MROPE, 1, 1, 2, 2, (1, 0, 0, 0)),
]


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("mode,n,heads,dim,n_dims,sections", ROPE_CASES)
def test_rope_axes(ctx, backend, mode, n, heads, dim, n_dims, sections, dtype, back):
    rng = np.random.default_rng(n * 100 + dim + mode)
    x = rng.standard_normal((n, heads, dim)).astype(np.float16 if dtype == "f16" else np.float32)
    pos = positions(n, rng)
    tx, tp = ctx.new_tensor(dtype, dim, heads, n), ctx.new_tensor("i32", 4 * n)
    turn = ctx.rope_multi_back if back else ctx.rope_multi
    y = run(ctx, backend, [turn(tx, tp, None, n_dims, sections, mode, 8192, 1e6)], [(tx, x), (tp, pos)])[0].reshape(n, heads, dim)
    want, mag = ref.rope(x.astype(np.float64), pos, mode, n_dims, sections, 1e6, back=back)
    bound = 10 * EPS32 * mag + (EPS16 * np.abs(want) + 2.0 ** -25 if dtype == "f16" else 0)
    assert np.all(np.abs(y - want) <= bound), np.max(np.abs(y - want) / (bound + 1e-30))


@pytest.mark.parametrize("mode", [MROPE, IMROPE, VISION])
def test_rope_axes_factors_and_yarn(ctx, backend, mode):
    """frequency factors, YaRN's ramp, a scale"""
    rng = np.random.default_rng(mode)
    n, heads, dim = 11, 3, 128
    n_dims = 64 if mode == VISION else 128
    x, pos = rng.standard_normal((n, heads, dim)).astype(np.float32), positions(n, rng, 5000)
    ff = (1 + rng.random(64)).astype(np.float32)
    tx, tp, tf = ctx.new_tensor("f32", dim, heads, n), ctx.new_tensor("i32", 4 * n), ctx.new_tensor("f32", 64)
    args = (n_dims, SECTIONS[mode], mode, 4096, 1e4, 0.25, 1.0, 0.9, 32.0, 1.0)
    outs = [ctx.rope_multi(tx, tp, tf, *args), ctx.rope_multi_back(tx, tp, tf, *args)]
    got = run(ctx, backend, outs, [(tx, x), (tp, pos), (tf, ff)])
    for y, back in zip(got, (False, True)):
        want, mag = ref.rope(x.astype(np.float64), pos, mode, n_dims, SECTIONS[mode], 1e4, ff, back, 4096, 0.25, 1.0, 0.9)
        # the ramp's 32-bit value is the definition's; one rounding of it apart moves a far angle by pos freq 2^-24
        bound = (10 * EPS32 + 5000 * EPS32) * mag
        assert np.all(np.abs(y.reshape(n, heads, dim) - want) <= bound)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("back", [False, True])
def test_rope_axes_strided(ctx, backend, dtype, back):
    """a view: heads inside wider rows at an odd offset (4- or 2-byte aligned), tokens apart"""
    rng = np.random.default_rng(3)
    n, heads, dim, wide = 6, 3, 64, 197
    t = np.float16 if dtype == "f16" else np.float32
    e = np.dtype(t).itemsize
    x, pos = rng.standard_normal((n, heads, wide)).astype(t), positions(n, rng)
    tx, tp = ctx.new_tensor(dtype, wide, heads, n), ctx.new_tensor("i32", 4 * n)
    view = ctx.view_4d(tx, dim, heads, n, 1, wide * e, wide * heads * e, wide * heads * n * e, 5 * e)
    turn = ctx.rope_multi_back if back else ctx.rope_multi
    y = run(ctx, backend, [turn(view, tp, None, dim, (8, 12, 12, 0), MROPE, 8192, 1e4)], [(tx, x), (tp, pos)])[0].reshape(n, heads, dim)
    want, mag = ref.rope(x[..., 5:5 + dim].astype(np.float64), pos, MROPE, dim, (8, 12, 12, 0), 1e4, back=back)
    assert np.all(np.abs(y - want) <= 10 * EPS32 * mag + (EPS16 * np.abs(want) + 2.0 ** -25 if dtype == "f16" else 0))


@pytest.mark.parametrize("mode", [NORMAL, NEOX])
@pytest.mark.parametrize("dtype,dim,n_dims", [("f32", 128, 128), ("f16", 128, 128), ("f32", 80, 60), ("f16", 20, 12)])
def test_rope_ext_back(ctx, backend, mode, dtype, dim, n_dims):
    """one axis: the gradient of rope_ext is the transposed rotation by the very same angles, so turning forth and
    back gives the input (cos^2 + sin^2 and two roundings a step), and both agree with the formula at near positions"""
    rng = np.random.default_rng(dim + mode)
    n, heads = 9, 4
    t = np.float16 if dtype == "f16" else np.float32
    x, pos = rng.standard_normal((n, heads, dim)).astype(t), np.arange(3, 3 + n, dtype=np.int32)
    tx, tp = ctx.new_tensor(dtype, dim, heads, n), ctx.new_tensor("i32", n)
    y = ctx.rope_ext(tx, tp, None, n_dims, mode, 8192, 1e4)
    z, b = ctx.rope_ext_back(y, tp, None, n_dims, mode, 8192, 1e4), ctx.rope_ext_back(tx, tp, None, n_dims, mode, 8192, 1e4)
    _, gz, gb = [a.reshape(n, heads, dim) for a in run(ctx, backend, [y, z, b], [(tx, x), (tp, pos)])]
    want, mag = ref.rope(x.astype(np.float64), pos[None], mode, n_dims, base=1e4, back=True)
    half = (EPS16 if dtype == "f16" else 0)
    # the 32-bit recurrence theta *= scale: (i + 2) half steps of an angle of at most 12
    assert np.all(np.abs(gb - want) <= (10 + 12 * (n_dims // 2 + 2)) * EPS32 * mag + half * np.abs(want) + (2.0 ** -25 if half else 0))
    assert np.all(np.abs(gz - x.astype(np.float64)) <= 2 * (20 * EPS32 + 2 * half) * np.maximum(mag, np.abs(x)) + (2.0 ** -23 if half else 0))


@pytest.mark.parametrize("mode", [MROPE, IMROPE, VISION])
def test_rope_axes_gradient_by_differences(ctx, backend, mode):
    """d <w, f(x)> / dx = f_back(w): central differences of the forward pass along random directions"""
    rng = np.random.default_rng(mode)
    n, heads, dim = 5, 2, 128
    n_dims = 64 if mode == VISION else 128
    x, w, d = (rng.standard_normal((n, heads, dim)).astype(np.float32) for _ in range(3))
    pos = positions(n, rng)
    a = [ctx.new_tensor("f32", dim, heads, n) for _ in range(3)]
    tp = ctx.new_tensor("i32", 4 * n)
    args = (tp, None, n_dims, SECTIONS[mode], mode, 8192, 1e4)
    h = np.float32(0.5)                                       # (the map is linear: any step is exact)
    up, down, g = run(ctx, backend, [ctx.rope_multi(a[0], *args), ctx.rope_multi(a[1], *args), ctx.rope_multi_back(a[2], *args)],
                      [(a[0], x + h * d), (a[1], x - h * d), (a[2], w), (tp, pos)])
    lhs = np.sum(w.astype(np.float64) * (up.reshape(x.shape).astype(np.float64) - down.reshape(x.shape)))
    rhs = np.sum(g.reshape(x.shape).astype(np.float64) * d)
    assert abs(lhs - rhs) <= 12 * EPS32 * 4 * np.sum(np.abs(w)) + 12 * EPS32 * 2 * np.sum(np.abs(d))


# ---- CONCAT --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "i32", "i64", "i8"])
@pytest.mark.parametrize("ne_a,dim,more", [((8, 3, 2, 1), 0, 4), ((512, 1, 7, 1), 0, 64), ((5, 3, 2, 2), 1, 1), ((5, 3, 2, 2), 2, 3), ((16, 2, 1, 3), 3, 2), ((7, 1, 1, 1), 0, 1)])
def test_concat(ctx, backend, dtype, ne_a, dim, more):
    rng = np.random.default_rng(more)
    np_t = {"f32": np.float32, "f16": np.float16, "i32": np.int32, "i64": np.int64, "i8": np.int8}[dtype]
    ne_b = tuple(more if i == dim else v for i, v in enumerate(ne_a))
    a, b = ((rng.standard_normal(ne[::-1]) * 50).astype(np_t) for ne in (ne_a, ne_b))
    ta, tb = ctx.new_tensor(dtype, *ne_a), ctx.new_tensor(dtype, *ne_b)
    y = run(ctx, backend, [ctx.concat(ta, tb, dim)], [(ta, a), (tb, b)])[0]
    assert np.array_equal(y, np.concatenate([a, b], axis=3 - dim))


def test_concat_strided(ctx, backend):
    """operands seen through a transpose and a row view"""
    rng = np.random.default_rng(0)
    a, b = rng.standard_normal((6, 4)).astype(np.float32), rng.standard_normal((4, 9)).astype(np.float32)
    ta, tb = ctx.new_tensor("f32", 4, 6), ctx.new_tensor("f32", 9, 4)
    y = ctx.concat(ctx.transpose(ta), ctx.view_4d(tb, 5, 4, 1, 1, 36, 144, 144, 8), 0)
    assert np.array_equal(run(ctx, backend, [y], [(ta, a), (tb, b)])[0][0, 0], np.concatenate([a.T, b[:, 2:7]], 1))


# ---- cache rows appended with the rotation on the way -------------------------------------------------
def decode_rows(raw, type_, width):
    """cache bytes -> values"""
    if type_ in ("f32", "f16"):
        return raw.view(np.float32 if type_ == "f32" else np.float16).reshape(-1, width).astype(np.float64)
    if type_ == "bf16":
        return (raw.view(np.uint16).astype(np.uint32) << 16).view(np.float32).reshape(-1, width).astype(np.float64)
    size = 34 if type_ == "q8_0" else 18
    b = raw.reshape(-1, width // 32, size)
    d = b[..., :2].copy().view(np.float16).astype(np.float64)
    q = b[..., 2:]
    v = q.copy().view(np.int8).astype(np.float64) if type_ == "q8_0" else np.concatenate([q & 15, q >> 4], -1).astype(np.float64) - 8
    return (d * v).reshape(-1, width)


HALF = {"f32": 0.0, "f16": EPS16, "bf16": EPSBF}


def cache_bytes(type_, width, rows, rng):
    v = rng.standard_normal((rows, width)).astype(np.float32)
    if type_ == "f32":
        return v.view(np.uint8).reshape(-1)
    if type_ == "f16":
        return v.astype(np.float16).view(np.uint8).reshape(-1)
    if type_ == "bf16":
        return (v.view(np.uint32) >> 16).astype(np.uint16).view(np.uint8).reshape(-1)
    size = 34 if type_ == "q8_0" else 18
    b = rng.integers(0, 256, (rows * width // 32, size), dtype=np.uint8)
    b[:, :2] = (rng.random((len(b), 1)) * 0.1).astype(np.float16).view(np.uint8)
    return b.reshape(-1)


def rope_node(ctx, x, pos, mode, dim, base=1e4):
    if mode in (NORMAL, NEOX):
        return ctx.rope_ext(x, pos, None, dim, mode, 8192, base)
    half = dim // 2
    sec = {MROPE: (half - 2 * (half * 3 // 8), half * 3 // 8, half * 3 // 8, 0), IMROPE: (half - 2 * (half * 5 // 16),) + 2 * (half * 5 // 16,) + (0,)}[mode]
    return ctx.rope_multi(x, pos, None, dim, sec, mode, 8192, base)


def rope_want(x, pos, mode, dim, base=1e4):
    half = dim // 2
    sec = {MROPE: (half - 2 * (half * 3 // 8), half * 3 // 8, half * 3 // 8, 0), IMROPE: (half - 2 * (half * 5 // 16),) + 2 * (half * 5 // 16,) + (0,)}.get(mode)
    return ref.rope(x.astype(np.float64), pos, mode, dim, sec or (1, 0, 0, 0), base)


def latent_graph(ctx, n, n_ctx, cache, mode, rope_first, idx="i64", rank=512, rot=64, keep=False):
    x, w = ctx.new_tensor("f32", rank + rot, n), ctx.new_tensor("f32", rank)
    pos = ctx.new_tensor("i32", n if mode in (NORMAL, NEOX) else 4 * n)
    kc, ix = ctx.new_tensor(cache, rank + rot, n_ctx), ctx.new_tensor(idx, n)
    row = 4 * (rank + rot)
    low = ctx.mul(ctx.rms_norm(ctx.view_4d(x, rank, n, 1, 1, row, row * n, row * n, 0), 1e-6), w)
    turned = rope_node(ctx, ctx.view_4d(x, rot, 1, n, 1, row, row, row * n, 4 * rank), pos, mode, rot)
    parts = [ctx.reshape(low, rank, 1, n), turned]
    if rope_first:
        parts.reverse()
    rows = ctx.reshape(ctx.concat(*parts, 0), rank + rot, n)
    return dict(x=x, w=w, pos=pos, cache=kc, idx=ix, low=low, rows=rows, out=ctx.set_rows(kc, rows, ix))


def latent_want(x, w, pos, mode, rope_first, rank=512):
    low = ref.rms_norm(x[:, :rank].astype(np.float64), w.astype(np.float64), float(np.float32(1e-6)))
    turned, mag = rope_want(x[:, None, rank:], pos, mode, x.shape[1] - rank)
    both, tol = [low, turned[:, 0]], [32 * EPS32 * np.abs(low), mag[:, 0]]
    if rope_first:
        both.reverse(), tol.reverse()
    return np.concatenate(both, 1), tol, low


@pytest.mark.parametrize("mode", [NORMAL, NEOX, MROPE, IMROPE])
@pytest.mark.parametrize("cache", ["f16", "bf16", "f32", "q8_0", "q4_0"])
@pytest.mark.parametrize("n,rope_first,idx", [(1, False, "i64"), (8, True, "i64"), (37, False, "i32")])
def test_append_latent(ctx, pkg, backend, mode, cache, n, rope_first, idx):
    rng = np.random.default_rng(n + mode)
    n_ctx = 64
    g = latent_graph(ctx, n, n_ctx, cache, mode, rope_first, idx)
    x, w = rng.standard_normal((n, 576)).astype(np.float32), (1 + 0.1 * rng.standard_normal(512)).astype(np.float32)
    pos = positions(n, rng, 40 if mode in (NORMAL, NEOX) else 30000)
    pos = pos[0] if mode in (NORMAL, NEOX) else pos
    cells = rng.permutation(n_ctx)[:n]
    before = cache_bytes(cache, 576, n_ctx, rng)
    graph = ctx.build(g["out"])
    ctx.alloc(backend)
    for t, a in ((g["x"], x), (g["w"], w), (g["pos"], pos), (g["idx"], cells.astype(np.int64 if idx == "i64" else np.int32)), (g["cache"], before)):
        t.set(a)
    backend.klog(True)
    ctx.compute(backend, graph)
    log = backend.klog_read()
    backend.klog(False)
    assert len(log) == 1 and log[0].startswith("append_rows norm=512"), log
    after = g["cache"].get_bytes()
    rest = np.setdiff1d(np.arange(n_ctx), cells)
    assert np.array_equal(after.reshape(n_ctx, -1)[rest], before.reshape(n_ctx, -1)[rest])      # the other cells as they were
    got = decode_rows(after, cache, 576)[cells]
    want, tol, _ = latent_want(x, w, pos if pos.ndim == 2 else pos[None], mode, rope_first)
    # one axis: (i + 2) half steps of the angle (below 41) from the 32-bit recurrence
    turn = (10 + (41 * 34 if mode in (NORMAL, NEOX) else 0)) * EPS32
    bound = np.concatenate([t * turn if t.shape[1] == 64 else t for t in tol], 1)
    if cache in HALF:
        assert np.all(np.abs(got - want) <= bound + HALF[cache] * (np.abs(want) + bound) + (2.0 ** -25 if cache == "f16" else 0))
    else:
        # a block's step is its largest magnitude / 127 (8: half a step each way; 4 bits: / 8, the far end clipped by
        # a whole step), known to 11 bits
        top = np.abs(want).reshape(n, 18, 32).max(-1, keepdims=True)
        lim = top / 127 * 0.5 + top * EPS16 if cache == "q8_0" else top / 8 + top * EPS16
        assert np.all(np.abs(got - want).reshape(n, 18, 32) <= lim * 1.001)


@pytest.mark.parametrize("cache", ["f16", "q8_0", "q4_0", "bf16"])
@pytest.mark.parametrize("mode", [NORMAL, NEOX, MROPE])
def test_append_fused_is_unfused(pkg, backend, cache, mode):
    """keys and values: the rows of the one launch are, bit for bit, those of ROPE and SET_ROWS one after the other"""
    rng = np.random.default_rng(5)
    n, heads, dim, n_ctx = 19, 4, 96, 40
    k, v = rng.standard_normal((n, heads, dim)).astype(np.float32), rng.standard_normal((n, heads * dim)).astype(np.float32)
    pos = positions(n, rng)
    pos = pos[0] if mode in (NORMAL, NEOX) else pos
    cells, before = rng.permutation(n_ctx)[:n].astype(np.int64), cache_bytes(cache, heads * dim, n_ctx, rng)
    seen = []
    for apart in (False, True):
        c = pkg.Context()
        tk, tv, tp = c.new_tensor("f32", dim, heads, n), c.new_tensor("f32", heads * dim, n), c.new_tensor("i32", len(pos.reshape(-1)))
        kc, vc, ix = c.new_tensor(cache, heads * dim, n_ctx), c.new_tensor("f16", heads * dim, n_ctx), c.new_tensor("i64", n)
        turned = rope_node(c, tk, tp, mode, dim)
        if apart:
            c.lib.mxg_set_output(turned.ptr)                  # its result is wanted: nothing may skip it
        outs = [c.set_rows(kc, c.reshape(turned, heads * dim, n), ix), c.set_rows(vc, tv, ix)]
        g = c.build(*outs)
        c.alloc(backend)
        for t, a in ((tk, k), (tv, v), (tp, pos), (kc, before), (vc, np.zeros((n_ctx, heads * dim), np.float16)), (ix, cells)):
            t.set(a)
        backend.klog(True)
        c.compute(backend, g)
        log = backend.klog_read()
        backend.klog(False)
        assert any(line.startswith("append_rows") for line in log) != apart, log
        seen.append((kc.get_bytes(), vc.get_bytes()))
        c.free()
    assert all(np.array_equal(a, b) for a, b in zip(*seen))
    assert np.array_equal(seen[0][1].view(np.float16).reshape(n_ctx, -1)[cells], v.astype(np.float16))


def test_append_keeps_what_others_read(ctx, backend):
    """the normalised part is read elsewhere too (a model's value path), and the row's other half is strided"""
    rng = np.random.default_rng(1)
    n = 6
    g = latent_graph(ctx, n, 16, "f16", MROPE, False)
    twice = ctx.scale(g["low"], 2.0)
    x, w, pos = rng.standard_normal((n, 576)).astype(np.float32), np.ones(512, np.float32), positions(n, rng)
    outs = run(ctx, backend, [g["out"], twice], [(g["x"], x), (g["w"], w), (g["pos"], pos), (g["idx"], np.arange(3, 3 + n)),
                                                (g["cache"], np.zeros((16, 576), np.float16))])
    want, _, low = latent_want(x, w, pos, MROPE, False)
    assert np.all(np.abs(outs[1].reshape(n, 512) - 2 * low) <= 64 * EPS32 * np.abs(low))
    assert rel(outs[0].reshape(16, 576)[3:3 + n], want) < 3e-4 and not outs[0].reshape(16, 576)[:3].any()


def test_append_outside_the_cache(ctx, backend):
    """a padded batch: tokens whose cell is outside the cache leave it as it was"""
    rng = np.random.default_rng(2)
    n, n_ctx = 5, 8
    g = latent_graph(ctx, n, n_ctx, "f16", NEOX, False)
    cells = np.array([2, -1, 7, n_ctx, 2 ** 40], np.int64)
    x, before = rng.standard_normal((n, 576)).astype(np.float32), rng.standard_normal((n_ctx, 576)).astype(np.float16)
    out = run(ctx, backend, [g["out"]], [(g["x"], x), (g["w"], np.ones(512, np.float32)), (g["pos"], np.arange(n, dtype=np.int32)), (g["idx"], cells),
                                         (g["cache"], before)])[0].reshape(n_ctx, 576)
    rest = [0, 1, 3, 4, 5, 6]
    assert np.array_equal(out[rest], before[rest]) and not np.array_equal(out[2], before[2]) and not np.array_equal(out[7], before[7])


@pytest.mark.parametrize("cache", ["f16", "f32"])
def test_append_to_one_cell(ctx, backend, cache):
    """several tokens of one cell: its values are theirs, each of one of them; the other cells are right"""
    rng = np.random.default_rng(3)
    n, n_ctx = 40, 16
    g = latent_graph(ctx, n, n_ctx, cache, NEOX, True)
    cells = np.full(n, 5, np.int64)
    cells[:3] = [0, 9, 15]
    x, w, pos = rng.standard_normal((n, 576)).astype(np.float32), np.ones(512, np.float32), np.arange(n, dtype=np.int32)
    before = np.zeros((n_ctx, 576), np.float32 if cache == "f32" else np.float16)
    out = run(ctx, backend, [g["out"]], [(g["x"], x), (g["w"], w), (g["pos"], pos), (g["idx"], cells), (g["cache"], before)])[0].reshape(n_ctx, 576)
    want = latent_want(x, w, np.broadcast_to(pos, (4, n)), NEOX, True)[0]
    off = np.abs(out[None, 5] - want[3:]).min(0)
    half = EPS16 if cache == "f16" else 64 * EPS32
    assert (off <= half * (1 + np.abs(want[3:]).max(0))).all()
    assert np.abs(out[[0, 9, 15]] - want[:3]).max() <= half * (1 + np.abs(want[:3]).max()) and not out[[1, 2, 3, 4, 6, 7, 8]].any()


# ---- attention whose keys are wider than its values -----------------------------------------------------
def quantise(x, type_):
    """values -> cache bytes whose values (decode_rows) are the reference's"""
    if type_ == "f16":
        return x.astype(np.float16).view(np.uint8).reshape(-1)
    b = x.reshape(-1, 32).astype(np.float64)
    if type_ == "q8_0":
        d = (np.abs(b).max(-1, keepdims=True) / 127).astype(np.float16)
        q = np.clip(np.round(b / np.where(d == 0, 1, d).astype(np.float64)), -128, 127).astype(np.int8).view(np.uint8)
    else:
        d = (np.abs(b).max(-1, keepdims=True) / -8).astype(np.float16)
        q = np.clip(np.round(b / np.where(d == 0, 1, d).astype(np.float64)) + 8, 0, 15).astype(np.uint8)
        q = q[:, :16] | (q[:, 16:] << 4)
    return np.concatenate([d.view(np.uint8), q], 1).reshape(-1)


def causal(S, n, m, lens=None):
    last = np.array(lens if lens is not None else [m] * S)[:, None] - n + np.arange(n)
    return np.where(np.arange(m) <= last[..., None], 0, -np.inf).astype(np.float16)[:, None]


class Case:
    """one attention call: data from a seed, the graph, the reference"""

    def __init__(self, ctx, form="latent", cache="f16", heads=4, kv_heads=1, n=1, m=64, S=1, kv_S=None, mask="causal", off=0, seed=0, scale=None, softcap=0.0,
                 max_bias=0.0, q_scale=1.0, spread=1.0):
        rng = np.random.default_rng(seed)
        dk, dv = (576, 512) if form == "latent" else (192, 128)
        kv_heads = kv_heads if form == "latent" else (kv_heads if kv_heads > 1 else heads)
        kv_S = kv_S or S
        self.q = (rng.standard_normal((S, n, heads, dk)) * q_scale).astype(np.float32)
        self.scale = scale if scale is not None else 192 ** -0.5
        self.raw = quantise(rng.standard_normal((kv_S, m, kv_heads, dk)) * spread, cache)
        self.k = decode_rows(self.raw, cache, dk).reshape(kv_S, m, kv_heads, dk).transpose(0, 2, 1, 3)
        tq = ctx.new_tensor("f32", dk, heads, n, S)
        tk = ctx.new_tensor(cache, dk, kv_heads, m, kv_S)
        kp = ctx.permute(tk, 0, 2, 1, 3)
        self.feeds = [(tq, self.q), (tk, self.raw)]
        if form == "latent":
            size = {"f16": 2, "q8_0": 34 / 32, "q4_0": 18 / 32}[cache]
            nb = kp.nb
            vp = ctx.view_4d(kp, dv, m, kv_heads, kv_S, nb[1], nb[2], nb[3], int(off * size))
            self.v = self.k[..., off:off + dv]
            self.tk, self.tv = tk, None
        else:
            v = rng.standard_normal((kv_S, m, kv_heads, dv)).astype(np.float16)
            self.v = v.astype(np.float64).transpose(0, 2, 1, 3)
            tv = ctx.new_tensor("f16", dv, kv_heads, m, kv_S)
            vp = ctx.permute(tv, 0, 2, 1, 3)
            self.feeds.append((tv, v))
            self.tk, self.tv = tk, tv
        self.mask = mask(rng, S, heads, n, m) if callable(mask) else causal(S, n, m) if mask == "causal" else None
        tm = None
        if self.mask is not None:
            ms = self.mask
            tm = ctx.new_tensor("f16", ms.shape[3], ms.shape[2], ms.shape[1], ms.shape[0])
            self.feeds.append((tm, ms))
        self.softcap, self.max_bias = softcap, max_bias
        self.out = ctx.flash_attn_ext(ctx.permute(tq, 0, 2, 1, 3), kp, vp, tm, self.scale, max_bias, softcap)
        self.shape = (S, n, heads, dv)
        self.ctx = ctx

    def want(self, **kw):
        return ref.attention(self.q.astype(np.float64).transpose(0, 2, 1, 3), self.k, self.v, self.mask, self.scale, self.max_bias, self.softcap, **kw)

    def run(self, backend, times=1):
        return run(self.ctx, backend, [self.out], self.feeds, times)[0].reshape(self.shape)


LATENT_SHAPES = [  # heads, n, m, S
    (4, 1, 1, 1), (16, 1, 63, 1), (32, 1, 64, 1), (32, 1, 65, 1), (10, 3, 300, 1), (32, 1, 1000, 3), (64, 1, 129, 2), (128, 1, 200, 1), (1, 1, 700, 1),
    (40, 17, 150, 1), (8, 33, 200, 2), (4, 100, 100, 1), (16, 40, 640, 1), (1, 70, 70, 1), (130, 64, 90, 1), (100, 10, 2000, 1), (128, 40, 1200, 1),
]


@pytest.mark.parametrize("cache", ["f16", "q8_0", "q4_0"])
@pytest.mark.parametrize("heads,n,m,S", LATENT_SHAPES)
def test_latent_attention(ctx, backend, cache, heads, n, m, S):
    c = Case(ctx, cache=cache, heads=heads, n=n, m=m, S=S, seed=heads + n + m)
    y = c.run(backend)
    assert np.isfinite(y).all() and rel(y, c.want()) < ATT_REL


@pytest.mark.parametrize("heads,kv_heads,n,m,S", [(4, 4, 1, 1, 1), (4, 4, 1, 333, 1), (4, 2, 20, 200, 1), (3, 3, 33, 64, 2), (8, 8, 5, 1200, 1), (8, 8, 130, 200, 1),
                                                  (2, 2, 300, 517, 1), (16, 16, 64, 96, 1), (1, 1, 257, 257, 1), (6, 2, 50, 31, 1), (520, 520, 65, 70, 1), (128, 64, 200, 230, 2)])
def test_expanded_attention(ctx, backend, heads, kv_heads, n, m, S):
    mask = "causal" if m >= n else lambda rng, S, H, n, m: np.zeros((1, 1, n, m), np.float16)
    c = Case(ctx, form="expanded", heads=heads, kv_heads=kv_heads, n=n, m=m, S=S, mask=mask, seed=heads + n + m)
    assert rel(c.run(backend), c.want()) < ATT_REL


def hidden_tiles(rng, S, H, n, m):
    """causal; whole tiles hidden at random, the first ones from most tokens, and single keys"""
    v = causal(S, n, m).copy()
    tiles = -(-m // 32)
    for t0 in range(0, n, 8):
        for t in np.nonzero(rng.random(tiles) < 0.4)[0]:
            v[:, :, t0:t0 + 8, 32 * t:32 * t + 32] = -np.inf
    v[:, :, n // 3:, :70] = -np.inf
    v[..., rng.random(m) < 0.02] = -np.inf
    return v


def window(rng, S, H, n, m):
    """the last 150 keys of each token, and nothing for one of them"""
    v = causal(S, n, m).copy()
    for t in range(n):
        v[:, :, t, :max(0, m - n + t - 150)] = -np.inf
    v[-1, :, n // 2] = -np.inf
    return v


@pytest.mark.parametrize("mask", ["causal", hidden_tiles, window], ids=["causal", "hidden_tiles", "window"])
@pytest.mark.parametrize("form,heads,n,m,S,cache", [("latent", 128, 80, 700, 1, "f16"), ("latent", 128, 30, 700, 2, "f16"), ("latent", 128, 62, 700, 1, "q8_0"),
                                                    ("latent", 128, 31, 650, 2, "q4_0"), ("latent", 8, 1000, 1000, 1, "f16"), ("latent", 8, 700, 700, 1, "q4_0"),
                                                    ("expanded", 64, 256, 600, 1, "f16"), ("expanded", 240, 20, 600, 1, "f16"), ("expanded", 128, 450, 450, 1, "f16")])
def test_many_tiles_a_workgroup(ctx, backend, form, heads, n, m, S, cache, mask):
    """enough rows that a workgroup walks 10 to 22 tiles: every slot of the rings several times, tiles listed from the mask's
    rows and from the map, some left out, the ones fetched before the list among them"""
    c = Case(ctx, form=form, heads=heads, n=n, m=m, S=S, cache=cache, mask=mask)
    assert rel(c.run(backend), c.want()) < ATT_REL


FORMS = [dict(form="latent", heads=8), dict(form="latent", heads=8, cache="q8_0"), dict(form="latent", heads=40), dict(form="latent", heads=40, cache="q4_0"),
         dict(form="expanded", heads=4), dict(form="expanded", heads=4, n=150, m=170),
         dict(form="latent", heads=128, n=70, m=110), dict(form="expanded", heads=512, n=66, m=80)]   # the variants of many rows


def sized(form, n=3, m=170):
    return {"n": n, "m": m, **form}


@pytest.mark.parametrize("form", FORMS)
def test_no_mask(ctx, backend, form):
    c = Case(ctx, mask=None, **sized(form))
    assert rel(c.run(backend), c.want()) < ATT_REL


@pytest.mark.parametrize("form", FORMS)
def test_one_cache_for_all_sequences(ctx, backend, form):
    c = Case(ctx, S=3, kv_S=1, **sized(form))
    assert rel(c.run(backend), c.want()) < ATT_REL


@pytest.mark.parametrize("form", FORMS)
def test_ragged_batch_and_a_free_slot(ctx, backend, form):
    """sequences of unequal length padded to one cache length, and one with nothing to look at: its rows are 0"""
    f = sized(form)
    lens = [f["m"], f["n"] + 2, 0]
    c = Case(ctx, S=3, mask=lambda rng, S, H, n, m: causal(S, n, m, lens), **f)
    y = c.run(backend)
    assert not y[2].any() and rel(y, c.want()) < ATT_REL


@pytest.mark.parametrize("form", FORMS)
def test_rows_the_mask_empties(ctx, backend, form):
    def mask(rng, S, H, n, m):
        v = np.where(rng.random((S, 1, n, m)) < 0.5, -np.inf, 0).astype(np.float16)
        v[:, :, ::2] = -np.inf
        return v
    c = Case(ctx, mask=mask, **sized(form))
    y = c.run(backend)
    assert not y[:, ::2].any() and rel(y, c.want()) < ATT_REL


@pytest.mark.parametrize("form", FORMS)
def test_mask_values(ctx, backend, form):
    """a bias, the type's lowest value beside zeros (weight 0), -inf; whole tiles of each"""
    def mask(rng, S, H, n, m):
        v = rng.standard_normal((S, 1, n, m)).astype(np.float16)
        v[..., rng.random(m) < 0.2] = -np.inf
        v[..., rng.random(m) < 0.2] = np.finfo(np.float16).min
        v[..., 64:128] = -np.inf
        v[..., 0] = 0
        return v
    c = Case(ctx, mask=mask, **sized(form))
    assert rel(c.run(backend), c.want()) < ATT_REL


@pytest.mark.parametrize("form", FORMS)
def test_rows_of_the_lowest_value(ctx, backend, form):
    """a row whose every key has the type's lowest value: the softmax of its scores, which 32 bits hold to 2^-9 beside
    65504 (weights off by 2^-9 of themselves each way, so results by 2^-8 of the largest value)"""
    def mask(rng, S, H, n, m):
        v = np.zeros((S, 1, n, m), np.float16)
        v[:, :, 0] = np.finfo(np.float16).min
        return v
    c = Case(ctx, mask=mask, **sized(form))
    y, want = c.run(backend), c.want()
    assert rel(y[:, 1:], want[:, 1:]) < ATT_REL and np.abs(y[:, 0] - want[:, 0]).max() <= 2.0 ** -8 * np.abs(c.v).max()


@pytest.mark.parametrize("form", FORMS)
def test_mask_of_every_head_bias_and_softcap(ctx, backend, form):
    def mask(rng, S, H, n, m):
        v = -np.abs(rng.standard_normal((S, H, n, m))).astype(np.float16)
        v[rng.random(v.shape) < 0.3] = -np.inf
        v[..., 0] = 0
        return v
    # the slope is a power in 32 bits: a few half steps of a bias below 8 move a score by 1e-6
    for kw in (dict(max_bias=8.0), dict(softcap=20.0)):
        c = Case(type(ctx)(), mask=mask, S=2, **kw, **sized(form))
        assert rel(c.run(backend), c.want()) < 2 * ATT_REL


@pytest.mark.parametrize("form", FORMS)
def test_what_masked_keys_hold(ctx, backend, form):
    """NaN and infinities in rows of the cache that the mask hides - for all queries, or for the earlier ones only"""
    f = sized(form)
    if f.get("cache", "f16") != "f16":
        pytest.skip("quantised rows hold no NaN but in a step")
    hidden = [5, 66, f["m"] - 1]

    def mask(rng, S, H, n, m):
        v = np.zeros((S, 1, n, m), np.float16)
        v[..., hidden] = -np.inf
        return v
    c = Case(ctx, mask=mask, **f)
    want = c.want()
    dk = c.k.shape[-1]
    raw = c.raw.view(np.float16).reshape(f["m"], -1, dk)
    raw[hidden[0]], raw[hidden[1]], raw[hidden[2]] = np.nan, np.inf, -np.inf
    c.feeds[1] = (c.feeds[1][0], raw)
    if c.tv is not None:
        v = c.feeds[2][1].copy()
        v.reshape(f["m"], -1)[hidden] = np.nan
        c.feeds[2] = (c.feeds[2][0], v)
    assert rel(c.run(backend), want) < ATT_REL


def test_a_nan_reaches_only_those_who_see_it(ctx, backend):
    c = Case(ctx, heads=4, n=20, m=20)
    want = c.want()
    raw = c.raw.view(np.float16).reshape(20, 576).copy()
    raw[12, 100] = np.nan
    c.feeds[1] = (c.feeds[1][0], raw)
    y = c.run(backend)
    assert rel(y[:, :12], want[:, :12]) < ATT_REL and np.isnan(y[:, 12:]).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("m", [100, 900])
def test_sinks(ctx, backend, form, m):
    """src[4]: a logit a head that joins the denominator (set as libllama does, on the node)"""
    f = sized(form, m=m)
    f["m"] = max(f["m"], f["n"])
    c = Case(ctx, **f)
    sinks = np.random.default_rng(9).standard_normal(f["heads"]).astype(np.float32) * 3
    ts = ctx.new_tensor("f32", f["heads"])
    c.out.raw.src[4] = ts.ptr
    c.feeds.append((ts, sinks))
    assert rel(c.run(backend), c.want(sinks=sinks)) < ATT_REL


@pytest.mark.parametrize("form,n,m", [("latent", 1, 40), ("latent", 3, 900), ("latent", 80, 900), ("expanded", 3, 40), ("expanded", 3, 900), ("expanded", 300, 900)])
def test_sinks_of_minus_infinity(ctx, backend, form, n, m):
    """add nothing, and leave a row that sees nothing 0: without splits, and with each of the joins"""
    def mask(rng, S, H, n, m):
        v = np.where(rng.random((S, 1, n, m)) < 0.3, -np.inf, 0).astype(np.float16)
        v[1, :, 0] = -np.inf
        return v
    c = Case(ctx, form=form, heads=8, n=n, m=m, S=2, mask=mask)
    ts = ctx.new_tensor("f32", 8)
    c.out.raw.src[4] = ts.ptr
    c.feeds.append((ts, np.full(8, -np.inf, np.float32)))
    y = c.run(backend)
    assert not y[1, 0].any() and rel(y, c.want()) < ATT_REL


@pytest.mark.parametrize("cache", ["f16", "q8_0", "q4_0"])
@pytest.mark.parametrize("heads,n,m", [(8, 2, 200), (64, 3, 150)])
def test_values_behind_the_rotated_channels(ctx, backend, cache, heads, n, m):
    c = Case(ctx, cache=cache, heads=heads, n=n, m=m, off=64)
    assert rel(c.run(backend), c.want()) < ATT_REL


@pytest.mark.parametrize("kv_heads", [2, 8])
def test_several_latent_heads(ctx, backend, kv_heads):
    c = Case(ctx, heads=16, kv_heads=kv_heads, n=9, m=140)
    assert rel(c.run(backend), c.want()) < ATT_REL


@pytest.mark.parametrize("q_scale,spread,scale", [(1e-6, 1.0, 5e4), (3e4, 1.0, 2e-6), (1e6, 1e-3, 5e-5), (1.0, 300.0, 2e-4)])
def test_magnitudes(ctx, backend, q_scale, spread, scale):
    """queries and keys far from 1 whose scores are O(1): the two terms follow the row's magnitude"""
    c = Case(ctx, heads=16, n=2, m=300, q_scale=q_scale, spread=spread, scale=scale)
    assert rel(c.run(backend), c.want()) < ATT_REL


@pytest.mark.parametrize("cache", ["q8_0", "q4_0"])
@pytest.mark.parametrize("spread", [1e-4, 40.0, 2e4])   # (2e5 would pass f16's range in a 4-bit step)
def test_magnitudes_of_steps(ctx, backend, cache, spread):
    """quantised rows far from 1, and rows whose steps differ by thousands: the first tiles small, later ones large"""
    c = Case(ctx, cache=cache, heads=16, n=2, m=300, spread=spread, scale=192 ** -0.5 / spread)
    assert rel(c.run(backend), c.want()) < ATT_REL
    c = Case(type(ctx)(), cache=cache, heads=40, n=2, m=300, spread=np.repeat([1e-3, 1e-2, 1.0], 100)[None, :, None, None], scale=192 ** -0.5)
    assert rel(c.run(backend), c.want()) < ATT_REL


def test_sharp_scores(ctx, backend):
    """scores up to several hundred: one key takes all; a score of 300 has a half step of 1.5e-5 in 32 bits"""
    c = Case(ctx, heads=16, n=4, m=500, scale=4.0)
    assert rel(c.run(backend), c.want()) < 500 * EPS32 * 4


@pytest.mark.parametrize("form", FORMS)
def test_replayed_graph(ctx, backend, form):
    """the same graph again and again, new inputs between, other work between them"""
    c = Case(ctx, **sized(form))
    first = c.run(backend)
    g = ctx.build(c.out)
    want = c.want()
    rng = np.random.default_rng(4)
    for i in range(4):
        q = rng.standard_normal(c.q.shape).astype(np.float32) if i % 2 else c.q
        c.feeds[0][0].set(q)
        ctx.compute(backend, g)
        y = c.out.numpy().reshape(c.shape)
        if i % 2 == 0:
            assert np.array_equal(y, first)                   # no sum depends on an order
        else:
            keep, c.q = c.q, q
            assert rel(y, c.want()) < ATT_REL
            c.q = keep
    assert rel(first, want) < ATT_REL


def test_captured_graphs(pkg, backend):
    """graphs of enough nodes to be captured, replayed in turn: they share the stream's workspace. Smaller ones run as they are"""
    cases = []
    for i, kw in enumerate((dict(heads=32, m=3000), dict(heads=16, n=20, m=500, cache="q4_0"), dict(form="expanded", heads=8, n=40, m=300))):
        c = Case(pkg.Context(), seed=i, **kw)
        y = c.out
        for f in (2.0, 0.5, 4.0, 0.25):
            y = c.ctx.scale(y, f)
        c.y, c.big, c.small = y, c.ctx.build(y), c.ctx.build(c.out)
        c.ctx.alloc(backend)
        for t, a in c.feeds:
            t.set(a)
        cases.append(c)
    before = backend.stats()["graph_replay"]
    for c in cases:
        for _ in range(3):
            c.ctx.compute(backend, c.small)
        c.first = c.out.numpy().reshape(c.shape)
        assert rel(c.first, c.want()) < ATT_REL
    assert backend.stats()["graph_replay"] == before
    for i in range(6):
        for c in cases:
            if i % 2:
                c.ctx.compute(backend, c.small)
            c.ctx.compute(backend, c.big)
            assert np.array_equal(c.y.numpy().reshape(c.shape), c.first)
    assert backend.stats()["graph_replay"] >= before + 12          # (the first pass runs, the second may record)
    for c in cases:
        c.ctx.free()


def test_two_backends_at_once(pkg, backend):
    """two streams with a workspace each, their graphs queued before either is waited for"""
    other = pkg.Backend(0)
    cases = []
    for i, be in enumerate((backend, other)):
        c = Case(pkg.Context(), heads=32, n=2, m=3000, seed=i)
        g = c.ctx.build(c.out)
        c.ctx.alloc(be)
        for t, a in c.feeds:
            t.set(a)
        cases.append((c, g, be))
    for _ in range(4):
        for c, g, be in cases:
            c.ctx.compute_async(be, g)
    for c, g, be in cases:
        be.synchronize()
        assert rel(c.out.numpy().reshape(c.shape), c.want()) < ATT_REL
        c.ctx.free()
    other.free()


def test_long_cache(ctx, backend):
    """a cache whose byte offsets pass 32 bits: 4 million rows of 1152 bytes, of which the mask shows a few far apart"""
    m, heads = 4_000_000, 4
    rng = np.random.default_rng(0)
    tq, tk, tm = ctx.new_tensor("f32", 576, heads, 1), ctx.new_tensor("f16", 576, m), ctx.new_tensor("f16", m, 1)
    nb = tk.nb
    out = ctx.flash_attn_ext(ctx.permute(tq, 0, 2, 1, 3), ctx.view_4d(tk, 576, m, 1, 1, nb[1], nb[2], nb[3], 0),
                             ctx.view_4d(tk, 512, m, 1, 1, nb[1], nb[2], nb[3], 0), tm, 192 ** -0.5)
    g = ctx.build(out)
    ctx.alloc(backend)
    seen = np.array([0, 63, 64, 1_863_999, 2_000_000, 3_728_271, 3_999_935, m - 1])
    rows = rng.standard_normal((len(seen), 576)).astype(np.float16)
    for i, r in zip(seen, rows):                              # the rest stays what the allocation held
        ctx.lib.mxg_tensor_set(tk.ptr, r.ctypes.data, int(i) * 1152, 1152)
    mask = np.full(m, -np.inf, np.float16)
    mask[seen] = 0
    tm.set(mask)
    q = rng.standard_normal((1, heads, 576)).astype(np.float32)
    tq.set(q)
    ctx.compute(backend, g)
    want = ref.attention(q[None].astype(np.float64).transpose(0, 2, 1, 3), rows.astype(np.float64)[None, None], rows[:, :512].astype(np.float64)[None, None],
                         None, 192 ** -0.5)
    assert rel(out.numpy().reshape(1, 1, heads, 512), want) < ATT_REL


# ---- as they are used: append, then attend -----------------------------------------------------------
@pytest.mark.parametrize("cache", ["f16", "q8_0", "q4_0"])
def test_prompt_then_tokens(pkg, backend, cache):
    """a prompt, then single tokens: rows appended and attended in one graph each, against the cache's own values"""
    rng = np.random.default_rng(7)
    heads, n_ctx = 16, 96
    w = (1 + 0.1 * rng.standard_normal(512)).astype(np.float32)
    ctx = pkg.Context()
    held = ctx.new_tensor(cache, 576, n_ctx)
    ctx.alloc(backend)
    held.set(np.zeros(held.nbytes(), np.uint8))
    done = 0
    steps = {}
    for n in (40, 1, 1, 1, 5, 1):
        m = 64 if done + n <= 64 else 96
        if (n, m) not in steps:
            c = pkg.Context()
            x, tw, pos, ix = c.new_tensor("f32", 576, n), c.new_tensor("f32", 512), c.new_tensor("i32", 4 * n), c.new_tensor("i64", n)
            row = 4 * 576
            low = c.mul(c.rms_norm(c.view_4d(x, 512, n, 1, 1, row, row * n, row * n, 0), 1e-6), tw)
            turned = rope_node(c, c.view_4d(x, 64, 1, n, 1, row, row, row * n, 2048), pos, MROPE, 64)
            put = c.set_rows(held, c.reshape(c.concat(c.reshape(low, 512, 1, n), turned, 0), 576, n), ix)
            nb = held.nb
            k = c.view_4d(held, 576, m, 1, 1, nb[1], nb[2], nb[3], 0)
            q, mask = c.new_tensor("f32", 576, heads, n), c.new_tensor("f16", m, n)
            out = c.flash_attn_ext(c.permute(q, 0, 2, 1, 3), k, c.view_4d(held, 512, m, 1, 1, nb[1], nb[2], nb[3], 0), mask, 192 ** -0.5)
            g = c.build(put, out)
            c.alloc(backend)
            tw.set(w)
            steps[n, m] = (c, g, x, pos, ix, q, mask, out)
        c, g, x, pos, ix, q, mask, out = steps[n, m]
        xs, qs = rng.standard_normal((n, 576)).astype(np.float32), rng.standard_normal((n, heads, 576)).astype(np.float32)
        p = np.broadcast_to(np.arange(done, done + n, dtype=np.int32), (4, n)).copy()
        ms = causal(1, n, m, [done + n])
        for t, a in ((x, xs), (pos, p), (ix, np.arange(done, done + n)), (q, qs), (mask, ms)):
            t.set(a)
        c.compute(backend, g)
        done += n
        values = decode_rows(held.get_bytes(), cache, 576)
        want, tol, _ = latent_want(xs, w, p, MROPE, False)
        slack = {"f16": EPS16, "q8_0": 1 / 127, "q4_0": 1 / 7}[cache]
        assert np.abs(values[done - n:done] - want).max() <= slack * np.abs(want).max() and not values[done:].any()
        ref_out = ref.attention(qs[None].astype(np.float64).transpose(0, 2, 1, 3), values[None, None, :m], values[None, None, :m, :512], ms, 192 ** -0.5)
        assert rel(out.numpy().reshape(1, n, heads, 512), ref_out) < ATT_REL
    for s in steps.values():
        s[0].free()
    ctx.free()


def test_graph_with_a_refused_node(pkg, ctx, backend):
    """a node that lost its support after it was built (a shortened pos) fails the graph; the backend lives on"""
    x, pos = ctx.new_tensor("f32", 64, 2, 3), ctx.new_tensor("i32", 12)
    y = ctx.rope_multi(x, pos, None, 64, (8, 12, 12, 0), MROPE, 8192, 1e4)
    g = ctx.build(y)
    ctx.alloc(backend)
    pos.raw.ne[0] = 11
    for _ in range(2):
        with pytest.raises(RuntimeError):
            ctx.compute(backend, g)
    pos.raw.ne[0] = 12
    x.set(np.ones((3, 2, 64), np.float32))
    pos.set(np.zeros(12, np.int32))
    ctx.compute(backend, g)
    assert np.array_equal(y.numpy().reshape(3, 2, 64), np.ones((3, 2, 64), np.float32))


def test_kernel_choice(pkg, backend):
    """the rows of a workgroup go by the rows there are; more tokens than a few read the mask once for all heads"""
    for kw, want in ((dict(heads=16, n=1, m=600), "rows=32 "), (dict(heads=130, n=64, m=90), "rows=64 nsplit=1 "), (dict(heads=128, n=40, m=1200), "rows=64 nsplit=3 "),
                     (dict(heads=130, n=64, m=90, cache="q4_0"), "rows=32 "), (dict(heads=8, n=200, m=1024), "map=1"), (dict(heads=32, n=40, m=600), "map=0"),
                     (dict(form="expanded", heads=2, n=1, m=600), "rows=32 "), (dict(form="expanded", heads=2, n=100, m=600), "rows=64 "),
                     (dict(form="expanded", heads=512, n=66, m=80), "rows=128 nsplit=1 ")):
        c = Case(pkg.Context(), **kw)
        backend.klog(True)
        c.run(backend)
        log = backend.klog_read()
        backend.klog(False)
        assert any("fattn_wide" in line and want in line for line in log), log
        c.ctx.free()
