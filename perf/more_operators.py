"""The operators of a decoder or query head on an image's tokens, as cases that can be timed and compared.

Kinds of case:

* cross     attention of queries to an encoder's keys and values of another length, with lengths or a mask of the keys.
* prefix    attention of a batch whose sequences share a prefix: its keys and values have no batch, each sequence has some of
            its own behind them, and the new tokens see their predecessors.
* residual  the residual stream plus a block's normed, gated and scaled output, and the next block's norm of the sum.
"""

import math

import torch

own = False
DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one query a head over the tokens of a 1008 px image, as an attention pool has it: latency counts
        dict(name="cross 1x1x5184 16x64", kind="cross", batch=1, new=1, keys=5184, heads=16, kv=16, dim=64, layout="token",
             lens=False, mask=False, type="fp16"),
        # 18 queries of a tag tree over the tokens of 64 images of 448 px, 16 heads of 48
        dict(name="cross 64x18x1025 16x48", kind="cross", batch=64, new=18, keys=1025, heads=16, kv=16, dim=48,
             layout="token", lens=False, mask=False, type="fp16"),
        # a decoder's step for 64 images of several sizes: one token each, grouped heads, keys and values from one product
        dict(name="cross 64x1x1025 32+8x128 bf16", kind="cross", batch=64, new=1, keys=1025, heads=32, kv=8, dim=128,
             layout="packed", lens=True, mask=False, type="bf16"),
        # the tokens of 8 images at 448 px read those of the same images at 1008 px
        dict(name="cross 8x1025x5184 16x64", kind="cross", batch=8, new=1025, keys=5184, heads=16, kv=16, dim=64,
             layout="token", lens=False, mask=False, type="fp16"),
        # four texts of 1000 tokens on letterboxed images, whose border patches are masked
        dict(name="cross 4x1000x4097 32+8x128 bf16", kind="cross", batch=4, new=1000, keys=4097, heads=32, kv=8, dim=128,
             layout="packed", lens=False, mask=True, type="bf16"),
        # one token of one text behind a 448 px image: latency counts
        dict(name="prefix 1x1 1025+16 16x64", kind="prefix", batch=1, new=1, prefix=1025, keys=16, heads=16, kv=16, dim=64,
             lens=False, type="fp16"),
        # a step of 64 answers about one 1008 px image, of several lengths
        dict(name="prefix 64x1 5184+256 32+8x128", kind="prefix", batch=64, new=1, prefix=5184, keys=256, heads=32, kv=8,
             dim=128, lens=True, type="bf16"),
        # 32 prompts of 48 tokens about one 1008 px image, read at once
        dict(name="prefix 32x48 5184+48 16x64", kind="prefix", batch=32, new=48, prefix=5184, keys=48, heads=16, kv=16,
             dim=64, lens=False, type="fp16"),
        # a step of 256 sequences with a long instruction in common and their own caches of up to 1024 tokens
        dict(name="prefix 256x1 16384+1024 32+8x128", kind="prefix", batch=256, new=1, prefix=16384, keys=1024, heads=32,
             kv=8, dim=128, lens=True, type="bf16"),
        # a single row between two blocks: latency counts
        dict(name="residual 1x1024 rms", kind="residual", rows=1, width=1024, post="rms", pre="rms", gate="none", scale=1.0,
             type="fp16"),
        # EVA02-L's rows at 32 images, LayerNorm before and after, a gate a channel (layer scale)
        dict(name="residual 32800x1024 layer", kind="residual", rows=32800, width=1024, post="layer", pre="layer",
             gate="channel", scale=1.0, type="fp16"),
        # a long prompt of a wide decoder: RMS norms before and after, an odd number of tokens
        dict(name="residual 9001x4096 rms bf16", kind="residual", rows=9001, width=4096, post="rms", pre="rms", gate="none",
             scale=0.5, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8, 12, 16])
    return kv * rng.choice([1, 1, 2, 4, 8]) if kv < 12 else kv, kv


def draw(rng):
    kind = rng.choice(["cross", "cross", "prefix", "prefix", "residual"])
    t = rng.choice(["fp16", "bf16"])
    if kind == "residual":
        width = 8 * _log(rng, 8, 1024)
        return dict(kind=kind, rows=_log(rng, 1, min(32800, 36_000_000 // width)), width=width,
                    post=rng.choice(["none", "rms", "layer"]), pre=rng.choice(["none", "rms", "layer"]),
                    gate=rng.choice(["none", "channel", "row"]), scale=rng.choice([1.0, 0.5]), type=t)
    heads, kv = _heads(rng)
    dim = rng.choice([32, 48, 64, 64, 72, 80, 96, 128, 128])
    if kind == "cross":
        keys = _log(rng, 1, 8192)
        batch = _log(rng, 1, min(64, max(1, 250_000_000 // (keys * kv * dim))))
        new = _log(rng, 1, min(2048, max(1, 65_000_000_000 // (batch * heads * keys * dim))))
        return dict(kind=kind, batch=batch, new=new, keys=keys, heads=heads, kv=kv, dim=dim,
                    layout=rng.choice(["token", "packed", "head"]), lens=rng.random() < 0.3, mask=rng.random() < 0.3, type=t)
    batch, prefix = _log(rng, 1, 256), _log(rng, 1, 16384)
    new = 1 if rng.random() < 0.5 else _log(rng, 2, 128)
    new = min(new, max(1, 60_000_000_000 // (batch * heads * prefix * dim)))
    keys = new + _log(rng, 1, min(1024, max(1, 250_000_000 // (batch * kv * dim)))) - 1
    return dict(kind=kind, batch=batch, new=new, prefix=prefix, keys=keys, heads=heads, kv=kv, dim=dim,
                lens=rng.random() < 0.5, type=t)


# ---- inputs, from the seed alone ----


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, device=DEV, generator=g) * std


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) + 1)
    t = TYPES[case["type"]]
    s = dict(case)
    if case["kind"] == "residual":
        rows, c = case["rows"], case["width"]
        x = _randn(g, rows, c)
        x[:, torch.randperm(c, device=DEV, generator=g)[: max(1, c // 100)]] *= 20.0  # outlier channels of a residual stream
        s["x"], s["y"] = x.to(t), _randn(g, rows, c, std=0.5).to(t)
        for n in ("post", "pre"):
            s[n + "_gamma"] = None if case[n] == "none" else 1.0 + _randn(g, c, std=0.1)
            s[n + "_beta"] = _randn(g, c, std=0.1) if case[n] == "layer" else None
        gates = {"none": 0, "channel": 1, "row": rows}[case["gate"]]
        s["gate"] = _randn(g, gates, c, std=0.3).to(t) if gates else None
        s["x_out"] = torch.empty(rows, c, dtype=t, device=DEV)
        s["h"] = torch.empty(rows, c, dtype=t, device=DEV) if case["pre"] != "none" else None
        return s
    b, n, k, h, kv, d = (case[x] for x in ("batch", "new", "keys", "heads", "kv", "dim"))
    s["scale"] = 1.0 / math.sqrt(d)
    s["work"] = None
    s["out"] = torch.empty(b, n, h, d, dtype=t, device=DEV)
    layout = case.get("layout", "head")  # prefix: caches keep a head's rows together
    if layout == "packed":  # one product's rows: keys and values next to each other
        packed = _randn(g, b, k, 2, kv, d, std=1.2).to(t)
        s["k"], s["v"] = packed[:, :, 0], packed[:, :, 1]
    elif layout == "head":
        s["k"], s["v"] = (_randn(g, b, kv, k, d, std=1.2).to(t).transpose(1, 2) for _ in range(2))
    else:
        s["k"], s["v"] = (_randn(g, b, k, kv, d, std=1.2).to(t) for _ in range(2))
    s["q"] = _randn(g, b, n, h, d, std=1.2).to(t)
    if case["kind"] == "prefix":
        s["prefix_k"], s["prefix_v"] = (_randn(g, case["prefix"], kv, d, std=1.2).to(t) for _ in range(2))
        s["lens"] = torch.randint(n, k + 1, (b,), device=DEV, generator=g).int() if case["lens"] else None
        return s
    s["lens"] = torch.randint(k // 2, k + 1, (b,), device=DEV, generator=g).int() if case["lens"] else None
    s["mask"] = None
    if case["mask"]:  # the patches of a letterboxed image, row by row: a band of rows or of columns is real
        side = math.isqrt(k - 1) + 1
        at = torch.arange(k, device=DEV)
        line = torch.stack((at // side, at % side))[torch.randint(2, (b,), device=DEV, generator=g)]
        border = torch.randint(side // 3 + 1, (b, 1), device=DEV, generator=g)
        s["mask"] = (line >= border) & (line < side - border)
    return s


# ---- the plain form ----


def _attend(q, k, v, scale, seen):
    """q [N, rows, D], k and v [N, keys, D] in float32, seen [N, 1 or rows, keys] or None: softmax(scale q k) v, 0 where nothing
    is seen."""
    x = (q @ k.transpose(1, 2).contiguous()) * scale
    if seen is not None:
        x = torch.where(seen, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total == 0, torch.ones_like(total), total)


def _grouped(q, kv):
    """[B, L, H, D] -> [B * KV, G * L, D]: the rows that read one head of keys."""
    b, n, h, d = q.shape
    return q.float().view(b, n, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(b * kv, h // kv * n, d)


def _ungrouped(o, q, kv):
    b, n, h, d = q.shape
    return o.view(b, kv, h // kv, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, h, d).to(q.dtype)


def _rows(x):
    """[B, L, KV, D] -> [B * KV, L, D] in float32."""
    return x.float().transpose(1, 2).reshape(-1, x.size(1), x.size(3))


def _plain_cross(s):
    kv, keys = s["kv"], s["keys"]
    seen = None
    if s["lens"] is not None:
        seen = torch.arange(keys, device=DEV) < s["lens"][:, None]
    if s["mask"] is not None:
        seen = s["mask"] if seen is None else seen & s["mask"]
    if seen is not None:
        seen = seen[:, None].expand(-1, kv, -1).reshape(-1, 1, keys)
    return _ungrouped(_attend(_grouped(s["q"], kv), _rows(s["k"]), _rows(s["v"]), s["scale"], seen), s["q"], kv)


def _plain_prefix(s):
    b, n, kv, keys, p = s["batch"], s["new"], s["kv"], s["keys"], s["prefix"]
    q = s["q"]
    lens = torch.full((b,), keys, device=DEV) if s["lens"] is None else s["lens"]
    last = lens[:, None] - n + 1 + torch.arange(n, device=DEV)  # [B, L]: own keys that a query sees
    group = q.size(2) // kv
    x = [None, None]
    # all sequences' rows against the prefix at once, each sequence's against its own keys
    qg = _grouped(q, kv)
    qp = qg.view(b, kv, -1, q.size(3)).transpose(0, 1).reshape(kv, -1, q.size(3))
    pk, pv = (s[w].float().transpose(0, 1) for w in ("prefix_k", "prefix_v"))
    x[0] = (qp @ pk.transpose(1, 2).contiguous()).view(kv, b, group * n, p).transpose(0, 1).reshape(b * kv, group * n, p)
    x[1] = qg @ _rows(s["k"]).transpose(1, 2).contiguous()
    seen = torch.arange(keys, device=DEV) < last[:, :, None]
    seen = seen[:, None, None].expand(-1, kv, group, -1, -1).reshape(b * kv, group * n, keys)
    x[1] = torch.where(seen, x[1], torch.full_like(x[1], -math.inf))
    top = torch.maximum(x[0].amax(-1, keepdim=True), x[1].amax(-1, keepdim=True))
    e = [torch.exp((y - top) * s["scale"]) for y in x]
    total = e[0].sum(-1, keepdim=True) + e[1].sum(-1, keepdim=True)
    o = e[0].view(b, kv, group * n, p).transpose(0, 1).reshape(kv, b * group * n, p) @ pv
    o = o.view(kv, b, group * n, -1).transpose(0, 1).reshape(b * kv, group * n, -1) + e[1] @ _rows(s["v"])
    return _ungrouped(o / total, q, kv)


def _normed(x, norm, gamma, beta):
    if norm == "none":
        return x
    if norm == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gamma
    return x + beta if norm == "layer" else x


def _plain_residual(s):
    y = _normed(s["y"].float(), s["post"], s["post_gamma"], s["post_beta"]) * s["scale"]
    if s["gate"] is not None:
        y = y * s["gate"].float()
    x = s["x"].float() + y
    if s["pre"] == "none":
        return x.to(s["x"].dtype)
    return x.to(s["x"].dtype), _normed(x, s["pre"], s["pre_gamma"], s["pre_beta"]).to(s["x"].dtype)


# ---- one pass ----


def run(s):
    if not own:
        return {"cross": _plain_cross, "prefix": _plain_prefix, "residual": _plain_residual}[s["kind"]](s)
    from foidfinder_amd import kernels as ops

    if s["kind"] == "residual":
        norms = {"none": ops.NORM_NONE, "rms": ops.NORM_RMS, "layer": ops.NORM_LAYER}
        ops.residual_norm(s["x"], s["y"], s["x_out"], s["h"], norms[s["post"]], s["post_gamma"], s["post_beta"],
                          norms[s["pre"]], s["pre_gamma"], s["pre_beta"], s["gate"], s["scale"], 1e-6)
        return s["x_out"] if s["h"] is None else (s["x_out"], s["h"])
    if s["kind"] == "cross":
        if s["work"] is None:  # the workspace that a program keeps
            s["work"] = torch.empty(ops.cross_attention_work(s["q"], s["k"]), dtype=torch.float32, device=DEV)
        ops.cross_attention(s["q"], s["k"], s["v"], s["out"], s["scale"], s["lens"], s["mask"], s["work"])
    else:
        if s["work"] is None:
            s["work"] = torch.empty(ops.prefix_attention_work(s["q"], s["prefix_k"], s["k"]), dtype=torch.float32, device=DEV)
        ops.prefix_attention(s["q"], s["prefix_k"], s["prefix_v"], s["k"], s["v"], s["out"], s["scale"], s["lens"], s["work"])
    return s["out"]


def work(case):
    if case["kind"] == "residual":
        rows, c = case["rows"], case["width"]
        moved = 2 * rows * c * (3 if case["pre"] == "none" else 4)
        moved += 2 * c * {"none": 0, "channel": 1, "row": rows}[case["gate"]]
        for n in ("post", "pre"):
            moved += 4 * c * {"none": 0, "rms": 1, "layer": 2}[case[n]]
        return {"bytes": moved, "flops": 14 * rows * c}
    b, n, k, h, kv, d = (case[x] for x in ("batch", "new", "keys", "heads", "kv", "dim"))
    q_and_out = 4 * b * n * h * d
    if case["kind"] == "prefix":
        mean = (n + k) / 2 if case["lens"] else k  # of the own keys' lengths
        seen = max(1.0, mean - (n - 1) / 2)  # of a query among them
        return {"bytes": q_and_out + 4 * kv * d * (case["prefix"] + b * mean), "flops": 4 * b * n * h * d * (case["prefix"] + seen)}
    share = 1.0
    if case["lens"]:
        share *= 0.75
    if case["mask"]:
        share *= 2 / 3  # borders of 0 to a third on two sides
    return {"bytes": q_and_out + 4 * b * kv * d * k * share, "flops": 4 * b * n * h * d * k * share}


# ---- the operators' definitions in 64 bits ----


def _softmax64(q, k, v, scale, hidden=None):
    """q [L, H, D], k and v [keys, KV, D] of what may be seen, hidden [L, keys] or None -> [L, H, D]."""
    group = q.size(1) // k.size(1)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    if k.size(0) == 0:
        return out
    for h in range(k.size(1)):
        kh, vh = k[:, h].double(), v[:, h].double()
        x = q[:, h * group : (h + 1) * group].double().reshape(-1, q.size(2)).matmul(kh.t()) * scale
        if hidden is not None:
            x = x.masked_fill(hidden.repeat_interleave(group, 0), -math.inf)
        out[:, h * group : (h + 1) * group] = torch.softmax(x, -1).matmul(vh).view(q.size(0), group, -1)
    return out


def _norm64(x, norm, gamma, beta):
    if norm == "none":
        return x
    if norm == "layer":
        centred = x - x.mean(1, keepdim=True)
        return centred * (centred.square().mean(1, keepdim=True) + 1e-6).rsqrt() * gamma.double() + beta.double()
    return x * (x.square().mean(1, keepdim=True) + 1e-6).rsqrt() * gamma.double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "residual":
        y = _norm64(s["y"].double(), s["post"], s["post_gamma"], s["post_beta"])
        gate = 1.0 if s["gate"] is None else s["gate"].double()
        x = s["x"].double() + case["scale"] * gate * y
        return x if case["pre"] == "none" else (x, _norm64(x, s["pre"], s["pre_gamma"], s["pre_beta"]))
    out = torch.empty(s["out"].shape, dtype=torch.float64, device=DEV)
    for b in range(case["batch"]):
        k, v = s["k"][b], s["v"][b]
        length = case["keys"] if s["lens"] is None else int(s["lens"][b])
        if case["kind"] == "prefix":
            n, p = case["new"], case["prefix"]
            k, v = torch.cat((s["prefix_k"], k[:length])), torch.cat((s["prefix_v"], v[:length]))
            place = torch.arange(p + length - n, p + length, device=DEV)
            out[b] = _softmax64(s["q"][b], k, v, s["scale"], torch.arange(p + length, device=DEV) > place[:, None])
            continue
        valid = torch.arange(length, device=DEV)
        if s["mask"] is not None:
            valid = valid[s["mask"][b, :length]]
        out[b] = _softmax64(s["q"][b], k[valid], v[valid], s["scale"])
    return out
