"""Latent attention over quantised caches whose blocks' steps differ by far: those beside V (the rotated channels) past what
f16 holds of them."""
import numpy as np
import pytest

from latent_ref import rel
from test_latent_gpu import ATT_REL, Case, decode_rows

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
