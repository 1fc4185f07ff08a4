"""Latent attention over quantised caches whose blocks' steps differ by far: those beside V (the rotated channels) past what
f16 holds of them, and large ones, there or in hidden keys, that the values' precision may not follow."""
import numpy as np
import pytest

from latent_ref import rel
from test_latent_gpu import ATT_REL, Case, decode_rows
from test_latent_weights_gpu import check, one_heavy_key

pytestmark = pytest.mark.gpu
SIZE = {"q8_0": 34, "q4_0": 18}


@pytest.fixture
def ctx(pkg):
    c = pkg.Context()
    yield c
    c.free()


def put_block(c, cache, keys, block, d, n):
    """the step d, and the whole numbers n (of one key, or all the same), in one block of these keys; K and V follow"""
    m = c.k.shape[2]
    c.raw = c.raw.copy()
    b = c.raw.reshape(m, 18, SIZE[cache])
    b[keys, block, :2] = np.array([d], np.float16).view(np.uint8)
    n = np.broadcast_to(n, 32).astype(np.int8)
    b[keys, block, 2:] = n.view(np.uint8) if cache == "q8_0" else ((n[:16] + 8) | (n[16:] + 8) << 4).astype(np.uint8)
    c.k = decode_rows(c.raw, cache, 576).reshape(c.k.shape)
    c.v = c.k[..., c.off:c.off + 512]
    c.feeds[1] = (c.feeds[1][0], c.raw)


@pytest.mark.parametrize("cache", ["q8_0", "q4_0"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("off,block", [(0, 17), (0, 16), (64, 1)])
@pytest.mark.parametrize("keys", ["one", "all", "every third"])
def test_steps_past_f16_beside_the_values(ctx, backend, cache, sign, off, block, keys):
    """a step of 100 in a block that only K has: scores of O(1) all the same, and every key keeps its weight"""
    c = Case(ctx, cache=cache, heads=16, n=2, m=300, off=off, mask=None)
    c.off = off
    c.q[..., 32 * block:32 * block + 32] = 1e-3 * np.abs(c.q[..., 32 * block:32 * block + 32])
    put_block(c, cache, {"one": [77], "all": slice(None), "every third": slice(1, None, 3)}[keys], block, 100.0, 3 * sign)
    assert rel(c.run(backend), c.want()) < ATT_REL


@pytest.mark.parametrize("cache", ["q8_0", "q4_0"])
@pytest.mark.parametrize("m,S,heads", [(32768, 1, 4), (2048, 256, 32)])
def test_a_large_step_beside_the_values(ctx, backend, cache, m, S, heads):
    """steps of 60 in a block that only K has, of a thousandth of that in V, and small weights: V's steps alone count"""
    c = one_heavy_key(ctx, "latent", cache, S, gap=8, heads=heads, n=1, m=m)
    c.off = 0
    c.q[..., 512:544] = 0
    put_block(c, cache, slice(1, None), 16, 60.0, 1)
    check(c, backend, 8)


@pytest.mark.parametrize("cache", ["q8_0", "q4_0"])
@pytest.mark.parametrize("m,S,heads", [(32768, 1, 4), (2048, 256, 32)])
def test_large_steps_of_hidden_keys(ctx, backend, cache, m, S, heads):
    """the same in V's blocks of keys that the mask hides, in the first tile of each split"""
    c = one_heavy_key(ctx, "latent", cache, S, gap=8, heads=heads, n=1, m=m)
    hidden = np.arange(5, m, 96)
    tm = ctx.new_tensor("f16", m, 1)
    c.mask = np.zeros((1, 1, 1, m), np.float16)
    c.mask[..., hidden] = -np.inf
    c.out.raw.src[3] = tm.ptr
    c.feeds.append((tm, c.mask))
    c.off = 0
    for block in (0, 9, 15):
        put_block(c, cache, hidden, block, 60.0, 5)
    check(c, backend, 8)


@pytest.mark.parametrize("shape", [dict(heads=4, n=1, m=20000), dict(heads=32, n=16, m=2000)])
@pytest.mark.parametrize("cache", ["q8_0", "q4_0"])
@pytest.mark.parametrize("block", [3, 10, 17])
@pytest.mark.parametrize("value", [np.inf, np.nan, 60.0, 100.0, -60000.0])
def test_one_step_of_a_hidden_key(ctx, backend, shape, cache, block, value):
    """a step of any size, or no number, in one block of a hidden key, on either half's side or beside V"""
    def mask(rng, S, H, n, m):
        v = np.zeros((S, 1, n, m), np.float16)
        v[..., [40, 700]] = -np.inf
        return v
    c = Case(ctx, cache=cache, mask=mask, **shape)
    want = c.want()
    c.raw = c.raw.copy()
    c.raw.reshape(-1, 18, SIZE[cache])[[40, 700], block, :2] = np.array([value], np.float16).view(np.uint8)
    c.feeds[1] = (c.feeds[1][0], c.raw)
    assert rel(c.run(backend), want) < ATT_REL


@pytest.mark.parametrize("cache", ["q8_0", "q4_0"])
@pytest.mark.parametrize("off", [0, 64])
def test_rows_of_zeros_first(ctx, backend, cache, off):
    """visible rows of zeros (steps of 0) in the first tiles of every split, and rows that see other keys than their neighbours"""
    def mask(rng, S, H, n, m):
        v = np.zeros((S, 1, n, m), np.float16)
        v[:, :, 1::2, 300:600] = -np.inf
        return v
    c = Case(ctx, cache=cache, mask=mask, heads=32, n=16, m=2000, off=off)
    c.off = off
    put_block(c, cache, slice(0, 400), slice(None), 0.0, 0)
    put_block(c, cache, slice(400, 600), 9, 50.0, 1)
    assert rel(c.run(backend), c.want()) < ATT_REL
