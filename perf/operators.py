"""The positions, the cache rows and the attention of models that keep one latent vector a token, as
cases to be timed: rotary positions with several axes (and their gradient), appending rotated rows to a
cache, attention over a latent cache (absorbed form), and attention with the keys and values expanded
from it. ``run`` computes a case in plain 32-bit torch operations, or, where ``own`` is set, with the
graph operators of libggml-mi355x.so.
"""
import math

import torch

own = False

RANK, ROT = 512, 64             # latent attention: channels of the latent vector, channels that carry the position
LATENT = RANK + ROT             # a cache row: the normalised latent vector, then the rotated channels
EK, EV = 192, 128               # the expanded form: channels of a key (128 + 64 rotated) and of a value
SCALE = 1.0 / math.sqrt(EK)     # both forms: scores are those of the expanded keys
EPS = 1e-6
MODES = {"axes": 8, "vision": 24, "interleaved": 40}
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK_BYTES = {"q8_0": 34, "q4_0": 18}      # of 32 values


def listed():
    return [
        # a vision-language model writes its answer: one token, the queries of 32 heads, three axes that agree
        {"name": "axes: one token", "op": "rope", "mode": "axes", "type": "f32", "back": False, "n": 1, "heads": 32, "dim": 128},
        # the vision tower: 39 x 39 patches of an image, 16 heads of 80 channels, rows and columns
        {"name": "axes: image patches", "op": "rope", "mode": "vision", "type": "f32", "back": False, "n": 1521, "heads": 16, "dim": 80},
        # fine-tuning on video: the gradient of 4096 positions' rotation, axes interleaved over the channels
        {"name": "axes: gradient, 4096", "op": "rope", "mode": "interleaved", "type": "f16", "back": True, "n": 4096, "heads": 32, "dim": 128},
        # serving: eight sequences, one new token each, into a shared latent cache
        {"name": "append: latent, 8 tokens", "op": "append", "form": "latent", "type": "f16", "n": 8, "n_ctx": 4096},
        # a prompt's ragged last part, 2011 latent rows
        {"name": "append: latent, prompt", "op": "append", "form": "latent", "type": "f16", "n": 2011, "n_ctx": 8192},
        # a 512-token micro-batch's keys (8 heads, rotated over three axes) and values
        {"name": "append: keys and values", "op": "append", "form": "axes", "type": "f16", "n": 512, "n_ctx": 4096, "heads": 8, "dim": 128},
        # the first steps of an answer: 32 heads against 256 latent rows
        {"name": "latent: decode, 256", "op": "latent", "cache": "f16", "heads": 32, "tok": 1, "seqs": 1, "n_kv": 256},
        # a batch of four long conversations of unequal length, padded to one cache length
        {"name": "latent: decode, 4 x 32768", "op": "latent", "cache": "f16", "heads": 32, "tok": 1, "seqs": 4, "n_kv": 32768},
        # the same over a cache held in 4 bits
        {"name": "latent: 4 bits, 4 x 32768", "op": "latent", "cache": "q4_0", "heads": 32, "tok": 1, "seqs": 4, "n_kv": 32768},
        # a 512-token micro-batch of a prompt against what is in the cache
        {"name": "latent: prompt, 512", "op": "latent", "cache": "f16", "heads": 32, "tok": 512, "seqs": 1, "n_kv": 4096},
        # the expanded form on a short ragged prompt
        {"name": "expanded: prompt, 499", "op": "expanded", "heads": 32, "tok": 499, "n_kv": 512},
        # the expanded form on the second half of a long prompt
        {"name": "expanded: prompt, 2048", "op": "expanded", "heads": 32, "tok": 2048, "n_kv": 4096},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {k: max(v) for k, v in _costs().items()}
    while True:
        op = rng.choice(["rope", "append", "latent", "latent", "expanded"])
        if op == "rope":
            mode = rng.choice(["axes", "vision", "interleaved"])
            c = {"op": op, "mode": mode, "type": rng.choice(["f32", "f16"]), "back": rng.random() < 0.5, "n": _log(rng, 1, 4096),
                 "heads": rng.choice([1, 2, 5, 8, 12, 16, 28, 32, 64]), "dim": rng.choice([64, 80, 128]) if mode == "vision" else rng.choice([64, 96, 128, 256])}
        elif op == "append":
            c = {"op": op, "form": rng.choice(["latent", "axes", "interleaved"]), "type": rng.choice(["f16", "bf16", "f32"]), "n": _log(rng, 1, 4096), "n_ctx": 8192}
            if c["form"] != "latent":
                c.update(heads=rng.choice([1, 2, 4, 8, 16]), dim=rng.choice([64, 80, 128]))
        elif op == "latent":
            tok = _log(rng, 1, 512) if rng.random() < 0.5 else rng.choice([1, 1, 1, 2, 3, 4])
            c = {"op": op, "cache": rng.choice(["f16", "f16", "q8_0", "q4_0"]), "heads": rng.choice([4, 10, 16, 32, 40, 64, 128]), "tok": tok,
                 "seqs": rng.choice([1, 1, 2, 3, 5]), "n_kv": _log(rng, tok, 32768)}
            c["idle"] = c["seqs"] > 1 and rng.random() < 0.25
        else:
            tok = _log(rng, 1, 2048)
            c = {"op": op, "heads": rng.choice([1, 4, 10, 16, 32, 64]), "tok": tok, "n_kv": tok + _log(rng, 1, 4096) - 1}
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return c


def _costs():
    every = [work(c) for c in listed()]
    return {k: [w[k] for w in every] for k in ("bytes", "flops")}


def work(case):
    c = case
    if c["op"] == "rope":
        e, size = c["n"] * c["heads"] * c["dim"], {"f32": 4, "f16": 2}[c["type"]]
        return {"bytes": 2 * e * size + 16 * c["n"], "flops": 3 * e}
    if c["op"] == "append":
        size = {"f32": 4, "f16": 2, "bf16": 2}[c["type"]]
        if c["form"] == "latent":
            return {"bytes": c["n"] * (LATENT * (4 + size) + 12) + 4 * RANK, "flops": c["n"] * (4 * RANK + 3 * ROT)}
        e = c["n"] * c["heads"] * c["dim"]
        return {"bytes": 2 * e * (4 + size) + c["n"] * 24, "flops": 3 * e}
    if c["op"] == "latent":
        row = 2 * LATENT if c["cache"] == "f16" else LATENT // 32 * BLOCK_BYTES[c["cache"]]
        lens = _lengths(c)
        pairs = sum(_pairs(c["tok"], n) for n in lens)
        rows = c["seqs"] * c["tok"] * c["heads"]
        return {"bytes": sum(lens) * row + rows * (LATENT + RANK) * 4 + c["seqs"] * c["tok"] * c["n_kv"] * 2, "flops": 2 * pairs * c["heads"] * (LATENT + RANK)}
    n = c["n_kv"]
    return {"bytes": c["heads"] * (n * (EK + EV) * 2 + c["tok"] * (EK + EV) * 4) + c["tok"] * n * 2, "flops": 2 * _pairs(c["tok"], n) * c["heads"] * (EK + EV)}


def _pairs(tok, n):
    """Key-query pairs that a causal mask leaves: the last `tok` of `n` positions ask."""
    return tok * n - tok * (tok - 1) // 2 if n else 0


def _lengths(c):
    """Tokens in the cache of each sequence of a batch: the first fills it, the others are shorter; the last of an
    `idle` case is a server's free slot, with nothing to look at."""
    lens = [max(c["tok"], c["n_kv"] - i * (c["n_kv"] // (2 * c["seqs"]))) for i in range(c["seqs"])]
    return lens[:-1] + [0] if c.get("idle") else lens


# ---- what a user's program holds before the call ----------------------------------------------------
def _sections(mode, dim):
    """Channel pairs of each axis (time, height, width, unused), as such models split them."""
    if mode == "vision":
        return [dim // 4, dim // 4, 0, 0]
    pairs = dim // 2
    if mode == "interleaved":
        side = pairs * 5 // 16
        return [pairs - 2 * side, side, side, 0]
    side = pairs * 3 // 8
    return [pairs - 2 * side, side, side, 0]


def _freqs(mode, dim, base):
    """Of every channel pair: which axis' position turns it, and by how much a step (64 bits)."""
    s = _sections(mode, dim)
    axis, power = [], []
    for i in range(dim // 2):
        k = i % sum(s)
        if mode == "interleaved":
            a = 1 if k % 3 == 1 and k < 3 * s[1] else 2 if k % 3 == 2 and k < 3 * s[2] else 0 if k % 3 == 0 and k < 3 * s[0] else 3
        else:
            a = 0 if k < s[0] else 1 if k < s[0] + s[1] else 2
        axis.append(a)
        power.append(k - sum(s[:a]) if mode == "vision" else i)
    n_dims = dim // 2 if mode == "vision" else dim
    return axis, [base ** (-2.0 * p / n_dims) for p in power]


def _positions(case, g):
    """int32 [4, n]: text counts on, an image's patches share the time and count rows and columns."""
    n = case["n"]
    if case.get("mode") == "vision":
        side = max(1, math.isqrt(n))
        i = torch.arange(n, device="cuda", dtype=torch.int32)
        return torch.stack([i // side, i % side, torch.zeros_like(i), torch.zeros_like(i)])
    start = int(torch.randint(0, 30000, (1,), generator=g, device="cuda"))
    i = torch.arange(n, device="cuda", dtype=torch.int32)
    image = (i // 64) % 2 == 1          # every other run of 64 tokens is an 8 x 8 image
    t = start + torch.where(image, i // 64 * 64, i)
    return torch.stack([t, t + torch.where(image, i % 64 // 8, 0), t + torch.where(image, i % 8, 0), torch.zeros_like(i)]).to(torch.int32)


def _quantise(x, kind):
    """[rows, n] float -> the bytes of its blocks of 32: a half-precision step, then 32 whole numbers of 8 or 4 bits."""
    b = x.float().reshape(x.shape[0], -1, 32)
    if kind == "q8_0":
        d = (b.abs().amax(-1, keepdim=True) / 127).half()
        q = torch.where(d > 0, (b / d.float()).round(), torch.zeros_like(b)).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    else:
        top = b.gather(-1, b.abs().argmax(-1, keepdim=True))
        d = (top / -8).half()
        q = torch.where(d != 0, (b / d.float()).round() + 8, torch.full_like(b, 8)).clamp(0, 15).to(torch.uint8)
        q = q[..., :16] | (q[..., 16:] << 4)
    return torch.cat([d.contiguous().view(torch.uint8), q], -1).reshape(x.shape[0], -1)


def _mask(tok, n_kv, lens):
    """Half precision [seqs, tok, n_kv]: 0 where a query may look, -inf elsewhere."""
    key = torch.arange(n_kv, device="cuda")
    last = torch.tensor(lens, device="cuda")[:, None] - tok + torch.arange(tok, device="cuda")[None]
    return torch.where(key[None, None] <= last[..., None], 0.0, -math.inf).half()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    c, s = case, {"case": case}
    if c["op"] == "rope":
        s["x"] = rand(c["n"], c["heads"], c["dim"]).to(DTYPE[c["type"]])
        s["pos"] = _positions(c, g)
        axis, freq = _freqs(c["mode"], c["dim"], 1e6)
        s["axis"], s["freq"] = torch.tensor(axis, device="cuda"), torch.tensor(freq, device="cuda", dtype=torch.float64)
    elif c["op"] == "append":
        latent = c["form"] == "latent"
        width = LATENT if latent else c["heads"] * c["dim"]
        s["pos"] = _positions(c, g)
        s["index"] = torch.randperm(c["n_ctx"], generator=g, device="cuda")[: c["n"]]     # cells are taken as they come free
        s["cache"] = rand(c["n_ctx"], width).to(DTYPE[c["type"]])
        axis, freq = _freqs("axes", ROT, 1e4) if latent else _freqs(c["form"], c["dim"], 1e6)
        s["axis"], s["freq"] = torch.tensor(axis, device="cuda"), torch.tensor(freq, device="cuda", dtype=torch.float64)
        if latent:
            s["x"], s["weight"] = rand(c["n"], LATENT), 1 + 0.1 * rand(RANK)
        else:
            s["k"], s["v"] = rand(c["n"], c["heads"], c["dim"]), rand(c["n"], c["heads"] * c["dim"])
            s["vcache"] = rand(c["n_ctx"], width).to(DTYPE[c["type"]])
    elif c["op"] == "latent":
        rows = rand(c["seqs"] * c["n_kv"], LATENT)
        s["q"] = rand(c["seqs"], c["tok"], c["heads"], LATENT)
        s["cache"] = rows.half() if c["cache"] == "f16" else _quantise(rows, c["cache"])
        s["cache"] = s["cache"].reshape(c["seqs"], c["n_kv"], -1)
        s["mask"] = _mask(c["tok"], c["n_kv"], _lengths(c))
    else:
        s["q"] = rand(c["tok"], c["heads"], EK)
        s["k"], s["v"] = rand(c["n_kv"], c["heads"], EK).half(), rand(c["n_kv"], c["heads"], EV).half()
        s["mask"] = _mask(c["tok"], c["n_kv"], [c["n_kv"]])
    if own:
        _graph(s)
    return s


# ---- the framework's operators ------------------------------------------------------------------------
_held = []


def _backend():
    """The package and one backend (a stream on the GPU), as a program keeps them."""
    if not _held:
        from mi355x_pkg import load_package
        pkg = load_package()
        _held.extend([pkg, pkg.Backend(0)])
    return _held


class _Memory:
    """A backend tensor's memory for torch; the tensor's context, which owns it, lives as long as a view does."""

    def __init__(self, t, shape, kind):
        self.owner = t.ctx
        self.__cuda_array_interface__ = {"data": (t.raw.data, False), "shape": tuple(shape), "typestr": kind, "version": 2}


def _torch_view(t, shape, dtype):
    """A backend tensor's memory as a torch tensor."""
    kind = {torch.float32: "<f4", torch.float16: "<f2", torch.bfloat16: "<i2", torch.uint8: "|u1", torch.int32: "<i4", torch.int64: "<i8"}[dtype]
    v = torch.as_tensor(_Memory(t, shape, kind), device="cuda")
    return v.view(torch.bfloat16) if dtype == torch.bfloat16 else v


def _graph(s):
    """The case's graph in backend memory, its inputs copied there from `s`; `s["out"]` are its outputs."""
    pkg, be = _backend()
    c, ctx, fill = s["case"], pkg.Context(), []

    def leaf(kind, value, *ne):
        t = ctx.new_tensor(kind, *ne)
        fill.append((t, value))
        return t

    if c["op"] == "rope":
        n, h, d = c["n"], c["heads"], c["dim"]
        x, pos = leaf(c["type"], s["x"], d, h, n), leaf("i32", s["pos"], 4 * n)
        turn = ctx.rope_multi_back if c["back"] else ctx.rope_multi
        outs = [(turn(x, pos, None, d // 2 if c["mode"] == "vision" else d, _sections(c["mode"], d), MODES[c["mode"]], 32768, 1e6), (n, h, d), DTYPE[c["type"]])]
    elif c["op"] == "append":
        n, dt = c["n"], DTYPE[c["type"]]
        index = leaf("i64", s["index"], n)
        if c["form"] == "latent":
            x, pos = leaf("f32", s["x"], LATENT, n), leaf("i32", s["pos"], 4 * n)
            weight, cache = leaf("f32", s["weight"], RANK), leaf(c["type"], s["cache"], LATENT, c["n_ctx"])
            row = 4 * LATENT
            low = ctx.mul(ctx.rms_norm(ctx.view_4d(x, RANK, n, 1, 1, row, row * n, row * n, 0), EPS), weight)
            turned = ctx.rope_multi(ctx.view_4d(x, ROT, 1, n, 1, row, row, row * n, 4 * RANK), pos, None, ROT, _sections("axes", ROT), MODES["axes"], 32768, 1e4)
            rows = ctx.reshape(ctx.concat(ctx.reshape(low, RANK, 1, n), turned, 0), LATENT, n)
            outs = [(ctx.set_rows(cache, rows, index), s["cache"].shape, dt)]
        else:
            h, d = c["heads"], c["dim"]
            k, v = leaf("f32", s["k"], d, h, n), leaf("f32", s["v"], d * h, n)
            kc, vc = leaf(c["type"], s["cache"], d * h, c["n_ctx"]), leaf(c["type"], s["vcache"], d * h, c["n_ctx"])
            turned = ctx.rope_multi(k, leaf("i32", s["pos"], 4 * n), None, d, _sections(c["form"], d), MODES[c["form"]], 32768, 1e6)
            outs = [(ctx.set_rows(kc, ctx.reshape(turned, d * h, n), index), s["cache"].shape, dt), (ctx.set_rows(vc, v, index), s["vcache"].shape, dt)]
    elif c["op"] == "latent":
        h, n, m, q = c["heads"], c["tok"], c["n_kv"], c["seqs"]
        x = ctx.permute(leaf("f32", s["q"], LATENT, h, n, q), 0, 2, 1, 3)
        cache = leaf(c["cache"], s["cache"], LATENT, m, 1, q)
        nb = cache.nb
        values = ctx.view_4d(cache, RANK, m, 1, q, nb[1], nb[2], nb[3], 0)
        outs = [(ctx.flash_attn_ext(x, cache, values, leaf("f16", s["mask"], m, n, 1, q), SCALE), (q, n, h, RANK), torch.float32)]
    else:
        h, n, m = c["heads"], c["tok"], c["n_kv"]
        x = ctx.permute(leaf("f32", s["q"], EK, h, n), 0, 2, 1, 3)
        k, v = (ctx.permute(leaf("f16", s[a], d, h, m), 0, 2, 1, 3) for a, d in (("k", EK), ("v", EV)))
        outs = [(ctx.flash_attn_ext(x, k, v, leaf("f16", s["mask"], m, n), SCALE), (n, h, EV), torch.float32)]
    s["ctx"], s["graph"] = ctx, ctx.build(*[o[0] for o in outs])
    ctx.alloc(be)
    for t, value in fill:
        _torch_view(t, value.shape, value.dtype).copy_(value)
    s["out"] = [_torch_view(*o) for o in outs]
    torch.cuda.synchronize()


# ---- the same in plain operations ---------------------------------------------------------------------
def _turn(x, pos, axis, freq, paired, back=False):
    """x [n, heads, dim] with its channel pairs (i, i + paired) turned by pos[axis] * freq."""
    angle = pos.double()[axis].t() * freq                       # [n, pairs]: far positions need 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    sin = -sin if back else sin
    a, b = x.float()[..., :paired], x.float()[..., paired:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _values(cache, kind):
    """Cache rows in 32 bits."""
    if kind == "f16":
        return cache.float()
    b = cache.reshape(*cache.shape[:-1], LATENT // 32, BLOCK_BYTES[kind])
    d = b[..., :2].contiguous().view(torch.float16).float()
    q = b[..., 2:].contiguous()
    q = q.view(torch.int8).float() if kind == "q8_0" else torch.cat([q & 15, q >> 4], -1).float() - 8
    return (d * q).reshape(*cache.shape[:-1], LATENT)


def _attend(q, k, v, mask):
    """q [..., rows, a], k [..., keys, a], v [..., keys, b], mask [..., rows, keys] or one that broadcasts."""
    score = torch.matmul(q, k.transpose(-1, -2)) * SCALE + mask
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, 1.0, total)


def run(s):
    if own:
        s["ctx"].compute_async(_backend()[1], s["graph"])
        return s["out"]
    c = s["case"]
    if c["op"] == "rope":
        return [_turn(s["x"], s["pos"], s["axis"], s["freq"], c["dim"] // 2, c["back"]).to(s["x"].dtype)]
    if c["op"] == "append":
        if c["form"] == "latent":
            x, low = s["x"], s["x"][:, :RANK]
            low = low * torch.rsqrt(low.square().mean(-1, keepdim=True) + EPS) * s["weight"]
            turned = _turn(x[:, None, RANK:], s["pos"], s["axis"], s["freq"], ROT // 2)[:, 0]
            s["cache"][s["index"]] = torch.cat([low, turned], -1).to(s["cache"].dtype)
            return [s["cache"]]
        s["cache"][s["index"]] = _turn(s["k"], s["pos"], s["axis"], s["freq"], c["dim"] // 2).flatten(1).to(s["cache"].dtype)
        s["vcache"][s["index"]] = s["v"].to(s["vcache"].dtype)
        return [s["cache"], s["vcache"]]
    if c["op"] == "latent":
        k = _values(s["cache"], c["cache"])
        mask = s["mask"].float()[:, :, None].expand(-1, -1, c["heads"], -1).reshape(c["seqs"], -1, c["n_kv"])
        return [_attend(s["q"].reshape(c["seqs"], -1, LATENT), k, k[..., :RANK], mask).reshape(c["seqs"], c["tok"], c["heads"], RANK)]
    q, k, v = (s[a].float().transpose(0, 1).contiguous() for a in "qkv")
    return [_attend(q, k, v, s["mask"].float()).transpose(0, 1).contiguous()]


# ---- the definition, in 64 bits -----------------------------------------------------------------------
def exact(case, seed):
    """What `run` returns, from the definitions: rotation as a product of complex numbers, softmax as exp over its sum."""
    s, c = prepare(case, seed), case

    def turned(x, pos, dim, mode, base, sign=1):
        axis, freq = _freqs(mode, dim, base)
        unit = torch.empty(x.shape[0], dim // 2, dtype=torch.complex128, device="cuda")
        for i, (a, f) in enumerate(zip(axis, freq)):
            turn = sign * f * pos[a].double()
            unit[:, i] = torch.complex(torch.cos(turn), torch.sin(turn))
        z = torch.complex(x.double()[..., : dim // 2], x.double()[..., dim // 2:]) * unit[:, None]
        return torch.cat([z.real, z.imag], -1)

    if c["op"] == "rope":
        return [turned(s["x"], s["pos"], c["dim"], c["mode"], 1e6, -1 if c["back"] else 1)]
    if c["op"] == "append":
        cache = s["cache"].double()
        if c["form"] == "latent":
            low = s["x"][:, :RANK].double()
            low = s["weight"].double() * low / (low.pow(2).sum(-1, keepdim=True) / RANK + EPS).sqrt()
            cache.index_copy_(0, s["index"], torch.cat([low, turned(s["x"][:, None, RANK:], s["pos"], ROT, "axes", 1e4)[:, 0]], -1))
            return [cache]
        cache.index_copy_(0, s["index"], turned(s["k"], s["pos"], c["dim"], c["form"], 1e6).flatten(1))
        return [cache, s["vcache"].double().index_copy_(0, s["index"], s["v"].double())]
    if c["op"] == "latent":
        k = torch.empty(c["seqs"], c["n_kv"], LATENT, dtype=torch.float64, device="cuda")
        if c["cache"] == "f16":
            k.copy_(s["cache"])
        else:
            w = BLOCK_BYTES[c["cache"]]
            for b in range(LATENT // 32):
                block = s["cache"][..., b * w:(b + 1) * w].contiguous()
                step, data = block[..., :2].contiguous().view(torch.float16).double(), block[..., 2:].contiguous()
                for j in range(32):
                    n = data[..., j].view(torch.int8).double() if w == 34 else ((data[..., j % 16] >> (4 * (j // 16))) & 15).double() - 8
                    k[..., 32 * b + j] = step[..., 0] * n
        out = torch.zeros(c["seqs"], c["tok"], c["heads"], RANK, dtype=torch.float64, device="cuda")
        for i, length in enumerate(_lengths(c)):
            for t0 in range(0, c["tok"], 64):
                q = s["q"][i, t0:t0 + 64].double()
                e = torch.tensordot(q, k[i, :length], dims=([2], [1])) * SCALE
                beyond = torch.arange(length, device="cuda")[None] > (length - c["tok"] + torch.arange(t0, t0 + q.shape[0], device="cuda"))[:, None]
                e = torch.softmax(e.masked_fill(beyond[:, None], -math.inf), -1)
                out[i, t0:t0 + 64] = torch.tensordot(e, k[i, :length, :RANK], dims=([2], [0]))
        return [out]
    out = torch.empty(c["tok"], c["heads"], EV, dtype=torch.float64, device="cuda")
    beyond = torch.arange(c["n_kv"], device="cuda")[None] > (c["n_kv"] - c["tok"] + torch.arange(c["tok"], device="cuda"))[:, None]
    for h in range(c["heads"]):
        e = s["q"][:, h].double() @ s["k"][:, h].double().t() * SCALE
        out[:, h] = torch.softmax(e.masked_fill(beyond, -math.inf), -1) @ s["v"][:, h].double()
    return [out]
