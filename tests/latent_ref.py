"""64-bit references of the rotary positions with several axes, the rotated cache rows and the attention
whose keys are wider than its values, written from their formulas."""
import numpy as np

NORMAL, NEOX, MROPE, VISION, IMROPE = 0, 2, 8, 24, 40
EPS32, EPS16, EPSBF = 2.0 ** -24, 2.0 ** -11, 2.0 ** -8        # half a rounding step, relative


def rope_freqs(mode, n_dims, sections, base):
    """(axis, exponent) of every channel pair that turns, and its step per position."""
    pairs = n_dims if mode == VISION else n_dims // 2
    total = sum(sections)
    axis, freq = np.zeros(pairs, int), np.zeros(pairs)
    for i in range(pairs):
        k, e = i % total, i
        if mode == IMROPE:
            a = 3
            for cand in range(3):
                if k % 3 == cand and k < 3 * sections[cand]:
                    a = cand
        else:
            a = int(np.searchsorted(np.cumsum(sections), k, side="right"))
            if mode == VISION:
                e = k - sum(sections[:a])
        axis[i], freq[i] = a, float(base) ** (-2.0 * e / n_dims)
    return axis, freq


def yarn(pairs, n_dims, base, n_ctx, fast, slow, freq_scale, ext, attn):
    """Frequency factor of each pair and the scale of cos and sin; the ramp in 32 bits, as the operator defines it."""
    f = np.float32
    if ext == 0:
        return np.full(pairs, float(f(freq_scale))), float(f(attn))

    def dim(rot):
        return f(n_dims) * np.log(f(n_ctx) / f(f(rot) * f(2) * f(np.pi))) / f(f(2) * np.log(f(base)))
    lo, hi = max(f(0), np.floor(dim(fast))), min(f(n_dims - 1), np.ceil(dim(slow)))
    y = (np.arange(pairs).astype(f) - f(lo)) / max(f(0.001), f(hi) - f(lo))
    mix = ((f(1) - np.minimum(f(1), np.maximum(f(0), y))) * f(ext)).astype(np.float64)
    return float(f(freq_scale)) * (1 - mix) + mix, float(f(attn)) * (1 + 0.1 * np.log(1 / float(f(freq_scale))))


def rope(x, pos, mode, n_dims, sections=(1, 0, 0, 0), base=10000.0, ff=None, back=False, n_ctx=8192, freq_scale=1.0, ext=0.0,
         attn=1.0, fast=32.0, slow=1.0):
    """x [tokens, heads, dim] float64; pos [axes, tokens]. Returns y and, element by element, the sum of the
    magnitudes of the pair it came from (for error bounds)."""
    n, heads, d = x.shape
    pairs = n_dims if mode == VISION else n_dims // 2
    if mode in (NORMAL, NEOX):
        axis, freq = np.zeros(pairs, int), float(base) ** (-2.0 * np.arange(pairs) / n_dims)
    else:
        axis, freq = rope_freqs(mode, n_dims, sections, base)
    factor, scale = yarn(pairs, n_dims, base, n_ctx, fast, slow, freq_scale, ext, attn)
    ang = np.asarray(pos, np.float64)[axis].T * freq * factor / (1.0 if ff is None else np.asarray(ff, np.float64)[:pairs])
    c, s = np.cos(ang)[:, None] * scale, np.sin(ang)[:, None] * scale * (-1 if back else 1)
    a = np.arange(pairs) * 2 if mode == NORMAL else np.arange(pairs)
    b = a + 1 if mode == NORMAL else a + pairs
    y, mag = x.copy(), np.abs(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    mag[..., a] = mag[..., b] = (np.abs(x[..., a]) + np.abs(x[..., b])) * scale
    return y, mag


def rms_norm(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def attention(q, k, v, mask=None, scale=1.0, max_bias=0.0, softcap=0.0, sinks=None):
    """q [S, H, n, DK], k [S or 1, Hkv, m, DK], v alike, mask [S or 1, H or 1, n, m]: [S, n, H, DV]."""
    S, H, n, _ = q.shape
    G = H // k.shape[1]
    out = np.zeros((S, n, H, v.shape[-1]))
    n2 = 1 << int(np.floor(np.log2(H)))
    for s in range(S):
        for h in range(H):
            kk, vv = k[s % k.shape[0], h // G], v[s % v.shape[0], h // G]
            e = q[s, h] @ np.where(np.isfinite(kk), kk, 0).T * scale
            if softcap:
                e = softcap * np.tanh(e / softcap)
            if mask is not None:
                slope = 1.0
                if max_bias:
                    slope = 2.0 ** (-max_bias / n2 * (h + 1)) if h < n2 else 2.0 ** (-max_bias / 2 / n2 * (2 * (h - n2) + 1))
                mm = mask[s % mask.shape[0], h % mask.shape[1]].astype(np.float64)
                e = np.where(np.isneginf(mm), -np.inf, e + slope * np.where(np.isneginf(mm), 0, mm))
            top = e.max(-1, keepdims=True)
            if sinks is not None:
                top = np.maximum(top, float(sinks[h]))
            top = np.where(np.isneginf(top), 0, top)
            p = np.exp(e - top)
            total = p.sum(-1, keepdims=True) + (np.exp(float(sinks[h]) - top) if sinks is not None else 0)
            out[s, :, h] = (p / np.where(total == 0, 1, total)) @ np.where(np.isfinite(vv), vv, 0)
    return out


def rel(x, ref):
    """2-norm of the difference over the 2-norm of the reference (0 when both are 0)."""
    d, r = np.linalg.norm(np.asarray(x, np.float64) - ref), np.linalg.norm(ref)
    return d / r if r else float(d)
