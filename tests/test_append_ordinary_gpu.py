"""Ordinary one-axis graphs (ROPE -> SET_ROWS of keys and of values) that the one launch for cache rows takes as well: each is,
bit for bit, what the nodes give one after the other."""
import numpy as np
import pytest

from latent_ref import MROPE, NEOX, NORMAL
from test_latent_gpu import cache_bytes

pytestmark = pytest.mark.gpu


def append(pkg, backend, apart, cache="f16", vcache=None, mode=NEOX, n=19, heads=4, dim=128, n_dims=None, ff=False, yarn=False, strided=False, idx="i64", far=30000,
           values=True, pad=0, one_cache=False):
    """the caches' bytes after one graph; `apart`: the rotation's result is an output, so nothing may skip it"""
    rng = np.random.default_rng(11)
    n_ctx, width, vcache = 40, heads * dim, vcache or cache
    c = pkg.Context()
    if strided:                                               # keys and values are parts of one projection's rows
        qkv = c.new_tensor("f32", 3 * width + 8, n)
        row = 4 * (3 * width + 8)
        k = c.view_4d(qkv, dim, heads, n, 1, 4 * dim, row, row * n, 4 * width)
        v = c.view_4d(qkv, width, n, 1, 1, row, row * n, row * n, 8 * width)
        feeds = [(qkv, rng.standard_normal((n, 3 * width + 8)).astype(np.float32))]
    else:
        k, v = c.new_tensor("f32", dim, heads, n), c.new_tensor("f32", width, n)
        feeds = [(k, rng.standard_normal((n, heads, dim)).astype(np.float32)), (v, rng.standard_normal((n, width)).astype(np.float32))]
    axes = 4 if mode == MROPE else 1
    pos, ix = c.new_tensor("i32", axes * n), c.new_tensor(idx, n)
    cells = rng.permutation(n_ctx)[:n]
    feeds += [(pos, rng.integers(0, far, axes * n).astype(np.int32)), (ix, cells.astype(np.int64 if idx == "i64" else np.int32))]
    tf = None
    if ff:
        tf = c.new_tensor("f32", dim // 2)
        feeds.append((tf, (1 + 7 * rng.random(dim // 2)).astype(np.float32)))
    args = (0.25, 1.0, 0.9, 32.0, 1.0) if yarn else ()
    nd = n_dims or dim
    turned = c.rope_multi(k, pos, tf, nd, (nd // 2 - 16, 8, 8, 0), mode, 4096, 1e4, *args) if mode == MROPE else c.rope_ext(k, pos, tf, nd, mode, 4096, 1e4, *args)
    if apart:
        c.lib.mxg_set_output(turned.ptr)
    big_k, big_v = c.new_tensor(cache, width + pad, n_ctx), c.new_tensor(vcache, width + pad, n_ctx)
    kc, vc = (c.view_4d(t, width, n_ctx, 1, 1, t.nb[1], t.nb[2], t.nb[3], 0) if pad else t for t in (big_k, big_v))
    feeds += [(big_k, cache_bytes(cache, width + pad, n_ctx, rng)), (big_v, cache_bytes(vcache, width + pad, n_ctx, rng))]
    outs = [c.set_rows(kc, c.reshape(turned, width, n), ix)]
    if values:
        outs.append(c.set_rows(kc if one_cache else vc, v, ix))
    g = c.build(*outs)
    c.alloc(backend)
    for t, a in feeds:
        t.set(a)
    backend.klog(True)
    c.compute(backend, g)
    log = backend.klog_read()
    backend.klog(False)
    out = big_k.get_bytes(), big_v.get_bytes()
    c.free()
    return out, [line for line in log if line.startswith("append_rows")]


CASES = [dict(), dict(mode=NORMAL), dict(mode=NORMAL, n=1), dict(n=1, heads=8), dict(n=33, heads=16), dict(n_dims=64), dict(mode=NORMAL, n_dims=32), dict(dim=80, n_dims=20),
         dict(ff=True), dict(mode=NORMAL, ff=True), dict(yarn=True), dict(mode=NORMAL, yarn=True, ff=True), dict(strided=True), dict(mode=NORMAL, strided=True, heads=3, dim=72),
         dict(idx="i32"), dict(values=False), dict(pad=32), dict(mode=NORMAL, pad=96, strided=True), dict(mode=MROPE, n_dims=64, yarn=True, ff=True), dict(heads=1, dim=64),
         dict(vcache="f32"), dict(mode=NORMAL, heads=64, dim=64), dict(heads=2, dim=256, far=1000000)]


@pytest.mark.parametrize("cache", ["f16", "f32", "q8_0", "q4_0"])
@pytest.mark.parametrize("kw", CASES)
def test_one_launch_is_node_by_node(pkg, backend, cache, kw):
    if cache[0] == "q" and kw.get("heads", 4) * kw.get("dim", 128) % 32:
        pytest.skip("rows of no whole blocks")
    (fused, log), (plain, none) = (append(pkg, backend, apart, cache, **kw) for apart in (False, True))
    assert len(log) == 1 and not none
    assert all(np.array_equal(a, b) for a, b in zip(fused, plain))


def test_keys_and_values_into_one_cache(pkg, backend):
    """the same cells twice: the values, which come second, are what stays"""
    (fused, log), (plain, _) = (append(pkg, backend, apart, one_cache=True) for apart in (False, True))
    assert len(log) == 1 and "v=0" in log[0]
    assert all(np.array_equal(a, b) for a, b in zip(fused, plain))
