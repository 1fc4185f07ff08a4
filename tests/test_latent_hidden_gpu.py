"""Latent attention over caches whose hidden keys hold infinities or NaN in a few channels only: two waves
hold a row's channels, so one of them may compute its half again beside one that does not."""
import numpy as np
import pytest

from latent_ref import rel
from test_latent_gpu import ATT_REL, Case

pytestmark = pytest.mark.gpu


@pytest.fixture
def ctx(pkg):
    c = pkg.Context()
    yield c
    c.free()


def hide(keys):
    """the mask that hides these keys from every row"""
    def mask(rng, S, H, n, m):
        v = np.zeros((S, 1, n, m), np.float16)
        v[..., keys] = -np.inf
        return v
    return mask


def blocks(c, cache):
    """the cache's bytes as [keys, 18, block], to be written in place"""
    c.raw = c.raw.copy()
    c.feeds[1] = (c.feeds[1][0], c.raw)
    return c.raw.reshape(-1, 18, {"q8_0": 34, "q4_0": 18}[cache])


def step(value):
    return np.array([value], np.float16).view(np.uint8)


# rows and splits: one row group of many splits, the 32-row and the 64-row kernel, 4 to 20 tiles a split
SPLIT = [dict(heads=4, n=1, m=20000), dict(heads=32, n=16, m=2000), dict(heads=128, n=40, m=1200)]


@pytest.mark.parametrize("shape", SPLIT)
@pytest.mark.parametrize("channel", [20, 300, 540])
@pytest.mark.parametrize("value", [np.inf, np.nan])
def test_one_channel_of_a_hidden_key(ctx, backend, shape, channel, value):
    """an infinity or a NaN in one channel of a hidden key: two waves hold a row's channels, one of them computes its half
    again, and both halves stay on one reference maximum"""
    c = Case(ctx, mask=hide([40, 700]), **shape)
    want = c.want()
    raw = c.raw.view(np.float16).reshape(-1, 576).copy()
    raw[[40, 700], channel] = value
    c.feeds[1] = (c.feeds[1][0], raw)
    assert rel(c.run(backend), want) < ATT_REL


@pytest.mark.parametrize("shape", SPLIT[:2])
@pytest.mark.parametrize("cache", ["q8_0", "q4_0"])
@pytest.mark.parametrize("block", [3, 10])
@pytest.mark.parametrize("value", [np.inf, np.nan])
def test_one_step_of_a_hidden_key(ctx, backend, shape, cache, block, value):
    """the same of a quantised cache: a step that is no number in one half's blocks"""
    c = Case(ctx, cache=cache, mask=hide([40, 700]), **shape)
    want = c.want()
    blocks(c, cache)[[40, 700], block, :2] = step(value)
    assert rel(c.run(backend), want) < ATT_REL


@pytest.mark.parametrize("cache", ["f16", "q8_0", "q4_0"])
@pytest.mark.parametrize("kw", [dict(softcap=20.0), dict(max_bias=8.0), dict(off=64)])
def test_recomputed_rows_take_every_term(ctx, backend, cache, kw):
    """softcap, ALiBi's slopes and values behind the rotated channels in rows that are computed again"""
    c = Case(ctx, cache=cache, mask=hide([40, 700]), heads=32, n=16, m=2000, **kw)
    want = c.want()
    if cache == "f16":
        raw = c.raw.view(np.float16).reshape(-1, 576).copy()
        raw[[40, 700], 400] = np.nan
        c.feeds[1] = (c.feeds[1][0], raw)
    else:
        blocks(c, cache)[[40, 700], 11, :2] = step(np.nan)
    assert rel(c.run(backend), want) < 2 * ATT_REL


def test_a_visible_infinity_of_no_weight(ctx, backend):
    """a visible key whose score is -inf has weight 0: the channels where its value is finite are those without it"""
    c = Case(ctx, heads=4, n=1, m=20000, mask=hide([]))
    c.q[..., 300] = -np.abs(c.q[..., 300])
    c.mask[..., 40] = -np.inf
    want = c.want()
    c.mask[..., 40] = 0
    raw = c.raw.view(np.float16).reshape(-1, 576).copy()
    raw[40, 300] = np.inf
    c.feeds[1] = (c.feeds[1][0], raw)
    y = c.run(backend)
    rest = np.arange(512) != 300
    assert np.isnan(y[..., 300]).all() and rel(y[..., rest], want[..., rest]) < ATT_REL
