"""Latent and expanded attention where one key (the first, as in most long contexts) outweighs every other by far, and its
value is small: the result is the rest of the cache, through thousands of weights of 2^-10 to 2^-22 of the largest.

Bounds. A score of 20 to base 2 is known to 2^-20 in 32 bits; the first key's enters as one product and four roundings, and
moves its share, and with it the whole result, by as much: 4 * 20 * 2^-24 beside the bound of scores of O(1)."""
import numpy as np
import pytest

from latent_ref import EPS32, rel
from test_latent_gpu import ATT_REL, Case, decode_rows, quantise

pytestmark = pytest.mark.gpu


@pytest.fixture
def ctx(pkg):
    c = pkg.Context()
    yield c
    c.free()


def one_heavy_key(ctx, form, cache, S, gap, **kw):
    """a case whose first key's score is `gap` (nats) above the mean of the others, whose scores spread by 0.6 to 0.9; S
    sequences share one cache. The last channel of K carries the gap alone. Values have a mean of 1, the first key's are small"""
    c = Case(ctx, form=form, cache=cache, S=S, kv_S=1, mask=None, **kw)
    dk, m = c.q.shape[-1], kw["m"]
    vw = 512 if form == "latent" else 128
    rng = np.random.default_rng(8)
    c.q *= np.float32(0.5)
    c.q[..., :vw] -= c.q[..., :vw].mean(-1, keepdims=True)      # (the values' mean moves no score)
    c.q[..., -1] = 8
    k = rng.standard_normal((m, dk))
    if form == "latent":
        k[:, :vw] += 1
    k[0] *= 0.01
    k[:, -1] = 0
    k[0, -1] = gap / (8 * c.scale)
    c.raw = quantise(k, cache)
    c.k = decode_rows(c.raw, cache, dk).reshape(1, 1, m, dk)
    c.feeds[1] = (c.feeds[1][0], c.raw)
    if form == "latent":
        c.v = c.k[..., :vw]
    else:
        v = (1 + rng.standard_normal((m, vw))).astype(np.float16)
        v[0] = (0.01 * v[0]).astype(np.float16)
        c.feeds[2] = (c.feeds[2][0], v)
        c.v = v.astype(np.float64).reshape(1, 1, m, vw)
    return c


def check(c, backend, gap, sink=-np.inf):
    y = c.run(backend)
    k, v = c.k[0, 0], c.v[0, 0]
    for s in (0, -1):                                           # (the first and the last sequence stand for the others)
        e = c.q[s].reshape(-1, k.shape[1]).astype(np.float64) @ k.T * c.scale
        if c.mask is not None:
            e[:, np.isneginf(c.mask[0, 0, 0])] = -np.inf
        top = np.maximum(e.max(-1, keepdims=True), sink)
        p = np.exp(e - top)
        want = p @ v / (p.sum(-1, keepdims=True) + np.exp(sink - top))
        assert rel(y[s].reshape(want.shape), want) < ATT_REL + 4 * (gap + 4) / np.log(2) * EPS32


# with the splits that the plan gives: one, but for few rows on a long cache
CASES = [("latent", "f16", dict(S=256, heads=64, n=1, m=4096)), ("latent", "f16", dict(S=256, heads=32, n=1, m=512)), ("latent", "f16", dict(S=1, heads=4, n=1, m=32768)),
         ("latent", "q8_0", dict(S=256, heads=32, n=1, m=2048)), ("latent", "q4_0", dict(S=256, heads=32, n=1, m=2048)),
         ("expanded", "f16", dict(S=512, heads=1, n=8, m=2048)), ("expanded", "f16", dict(S=500, heads=1, n=64, m=2048)),
         ("expanded", "f16", dict(S=512, heads=1, n=128, m=2048)), ("expanded", "f16", dict(S=1, heads=1, n=1, m=8192))]


@pytest.mark.parametrize("gap", [8, 11, 14])
@pytest.mark.parametrize("form,cache,kw", CASES)
def test_one_heavy_key(ctx, backend, form, cache, kw, gap):
    check(one_heavy_key(ctx, form, cache, gap=gap, **kw), backend, gap)


@pytest.mark.parametrize("form,cache,kw", [CASES[i] for i in (0, 1, 2, 3, 7)])
def test_a_sink_that_outweighs_the_keys(ctx, backend, form, cache, kw):
    """the same weight in a sink instead of a key: without splits and with the join"""
    c = one_heavy_key(ctx, form, cache, gap=0, **kw)
    sinks = np.full(kw["heads"], 11, np.float32)
    ts = ctx.new_tensor("f32", kw["heads"])
    c.out.raw.src[4] = ts.ptr
    c.feeds.append((ts, sinks))
    check(c, backend, 11, sink=11)


@pytest.mark.parametrize("form,cache,kw", [CASES[i] for i in (0, 1, 3, 5)])
def test_heavy_keys_one_after_another(ctx, backend, form, cache, kw):
    """every 40th key is heavier than the last: the reference maximum is raised again and again, from 0 to 36 nats"""
    c = one_heavy_key(ctx, form, cache, gap=0, **kw)
    m = kw["m"]
    k = c.k.reshape(m, -1).copy()
    k[::40, -1] = np.linspace(0, 36, len(k[::40])) / (8 * c.scale)
    c.raw = quantise(k, cache)
    c.k = decode_rows(c.raw, cache, k.shape[1]).reshape(1, 1, m, -1)
    if form == "latent":
        c.v = c.k[..., :512]
    c.feeds[1] = (c.feeds[1][0], c.raw)
    check(c, backend, 36)
