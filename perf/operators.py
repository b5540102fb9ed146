"""The operators around a 4-bit (MX) linear and a head-normed attention, as cases that can be timed and compared.

Kinds of case:

* quant    rows to MX4 codes (norm, rotation by blockdiag(H128), 4-bit codes with a shared exponent per 32 columns) and
           the codes back to the values that they stand for.
* gemm     the MX4 product of codes that are in hand with a fused epilogue (bias, residual, tanh GELU, SwiGLU).
* qk       norm of each head's queries and keys with the position rotation in the same pass.

An MX4 tensor of [T, C] is codes uint8 [T, C / 2] (two E2M1 codes a byte, the even column in the low half) and scale int32
[C / 128, T]: word [b, t] holds the exponents (E8M0, bias 127, 255 = not a number) of columns 128 b + 32 i of row t in byte i.
"""

import math

import torch

own = False
DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ROOT128 = 0.08838834764831845  # 1 / sqrt(128)
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # E2M1 magnitudes by code


def listed():
    return [
        # a single row before a 1024-wide linear: the call a one-token step or a pooled row makes, where latency counts
        dict(name="quant 1x1024 rms", kind="quant", rows=1, width=1024, real=1024, norm="rms", rotate=True, type="fp16"),
        # EVA02-L's rows before QKV and fc1 at 32 images: LayerNorm, rotation and codes in one pass
        dict(name="quant 32800x1024 layer", kind="quant", rows=32800, width=1024, real=1024, norm="layer", rotate=True,
             type="fp16"),
        # EVA02-L's hidden rows before fc2 (2730 real columns of 2816) at 5 images
        dict(name="quant 5125x2816 layer", kind="quant", rows=5125, width=2816, real=2730, norm="layer", rotate=True,
             type="fp16"),
        # PixAI's hidden rows of one 1008 px image, without a norm, in bf16
        dict(name="quant 5184x4736 bf16", kind="quant", rows=5184, width=4736, real=4736, norm="none", rotate=True,
             type="bf16"),
        # Haruka's QKV on a single row: the weights' stream and the launch are all there is
        dict(name="gemm 1x2304x768 bias", kind="gemm", rows=1, cols=2304, width=768, epi="bias", type="fp16"),
        # Haruka's tag head on 16 images: fp32 logits of 98 782 tags, bounded by reading the weights
        dict(name="gemm 16x98782x1152 fp32", kind="gemm", rows=16, cols=98782, width=1152, epi="bias", type="fp32"),
        # EVA02-L's fc2 at one image: few rows, a long K, the residual added
        dict(name="gemm 1025x1024x2816 residual", kind="gemm", rows=1025, cols=1024, width=2816, epi="residual",
             type="fp16"),
        # PixAI's fc1 on one 1008 px image: GELU, in bf16
        dict(name="gemm 5184x4736x1024 gelu bf16", kind="gemm", rows=5184, cols=4736, width=1024, epi="gelu", type="bf16"),
        # EVA02-L's fc1 at 32 images: the largest product, SwiGLU on column pairs
        dict(name="gemm 32800x5632x1024 swiglu", kind="gemm", rows=32800, cols=5632, width=1024, epi="swiglu", type="fp16"),
        # one new token of a grouped-query decoder: 32 query and 8 key heads of 128, split halves, its position given
        dict(name="qk 1x32+8x128 rms bf16", kind="qk", rows=1, heads=32, kv=8, dim=128, rot=128, norm="rms", pairs=False,
             packed=True, given=True, table=8192, type="bf16"),
        # EVA02-L's packed QKV rows at 32 images: 16 heads of 64, LayerNorm per head, neighbouring pairs
        dict(name="qk 32800x16+16x64 layer", kind="qk", rows=32800, heads=16, kv=16, dim=64, rot=64, norm="layer",
             pairs=True, packed=True, given=False, table=1025, type="fp16"),
        # a long prompt of a grouped-query decoder, an odd number of tokens
        dict(name="qk 9001x32+8x128 rms bf16", kind="qk", rows=9001, heads=32, kv=8, dim=128, rot=128, norm="rms",
             pairs=False, packed=True, given=True, table=16384, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quant", "gemm", "gemm", "qk"])
    if kind == "quant":
        width = 128 * _log(rng, 1, 48)
        norm = rng.choice(["none", "rms", "layer"])
        real = width if norm == "none" or rng.random() < 0.5 else max(1, width - rng.randint(0, 127))
        return dict(kind=kind, rows=_log(rng, 1, min(32800, 36_000_000 // width)), width=width, real=real, norm=norm,
                    rotate=rng.random() < 0.75, type=rng.choice(["fp16", "bf16"]))
    if kind == "gemm":
        width = 128 * _log(rng, 1, 40)
        epi = rng.choice(["bias", "residual", "gelu", "swiglu"])
        kind_of = rng.choice(["fp16", "fp16", "bf16", "fp32"] if epi == "bias" else ["fp16", "bf16"])
        cols = _log(rng, 16, 8192)
        if epi == "bias" and rng.random() < 0.2:  # a tag head: few rows, tens of thousands of columns
            return dict(kind=kind, rows=_log(rng, 1, 64), cols=_log(rng, 8192, 98782), width=128 * rng.randint(4, 10),
                        epi=epi, type="fp32")
        if epi == "swiglu":
            cols += cols % 2
        most = min(32800, 189_000_000_000 // (cols * width), 90_000_000 // cols)
        return dict(kind=kind, rows=_log(rng, 1, max(1, most)), cols=cols, width=width, epi=epi, type=kind_of)
    dim = rng.choice([64, 64, 80, 96, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 12, 16])
    heads = kv * rng.choice([1, 1, 2, 4]) if kv < 12 else kv
    rot = dim if rng.random() < 0.7 else 16 * rng.randint(1, dim // 16)
    given = rng.random() < 0.5
    return dict(kind=kind, rows=_log(rng, 1, min(32800, 60_000_000 // ((heads + kv) * dim))), heads=heads, kv=kv, dim=dim,
                rot=rot, norm=rng.choice(["none", "rms", "rms", "layer"]), pairs=rng.random() < 0.5,
                packed=rng.random() < 0.7, given=given, table=_log(rng, 1, 16384), type=rng.choice(["fp16", "bf16"]))


# ---- inputs, from the seed alone ----


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, device=DEV, generator=g) * std


def _codes(g, rows, width, std):
    """Codes and scales of normal values, as a rotation leaves them: made in slices, to bound the memory in flight."""
    codes = torch.empty(rows, width // 2, dtype=torch.uint8, device=DEV)
    scale = torch.empty(width // 128, rows, dtype=torch.int32, device=DEV)
    step = max(1, (1 << 25) // width)
    for r in range(0, rows, step):
        mag, sign, e = _encode(_randn(g, min(step, rows - r), width, std=std))
        c = mag + 8 * sign
        codes[r : r + step] = (c[:, 0::2] + 16 * c[:, 1::2]).to(torch.uint8)
        e = e.long().view(-1, width // 128, 4)
        word = e[..., 0] + (e[..., 1] << 8) + (e[..., 2] << 16) + (e[..., 3] << 24)
        scale[:, r : r + step] = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32).t()
    return codes, scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) + 1)
    t, rows = TYPES[case["type"]], case["rows"]
    s = dict(case)
    if case["kind"] == "quant":
        x = _randn(g, rows, case["width"])
        cols = torch.randperm(case["width"], device=DEV, generator=g)[: max(1, case["width"] // 100)]
        x[:, cols] *= 20.0  # 1 % of the channels are outliers, as in a residual stream
        x[:, case["real"] :] = 0
        s["x"] = x.to(t)
        gamma, beta = 1.0 + _randn(g, case["width"], std=0.02), _randn(g, case["width"], std=0.02)
        gamma[case["real"] :] = 0
        beta[case["real"] :] = 0
        s["gamma"] = None if case["norm"] == "none" else gamma
        s["beta"] = beta if case["norm"] == "layer" else None
        s["codes"] = torch.empty(rows, case["width"] // 2, dtype=torch.uint8, device=DEV)
        s["scale"] = torch.empty(case["width"] // 128, rows, dtype=torch.int32, device=DEV)
        s["out"] = torch.empty(rows, case["width"], dtype=t, device=DEV)
    elif case["kind"] == "gemm":
        n, k = case["cols"], case["width"]
        s["a"], s["a_scale"] = _codes(g, rows, k, 1.0)
        s["w"], s["w_scale"] = _codes(g, n, k, 1.0 / math.sqrt(k))
        s["bias"] = _randn(g, n, std=0.02)
        out_cols = n // 2 if case["epi"] == "swiglu" else n
        s["residual"] = _randn(g, rows, n).to(t) if case["epi"] == "residual" else None
        s["out"] = torch.empty(rows, out_cols, dtype=t, device=DEV)
    else:
        h, kv, d, r = case["heads"], case["kv"], case["dim"], case["rot"]
        wide = h + 2 * kv if case["packed"] else h + kv  # packed rows hold the values too
        x = _randn(g, rows, wide, d, std=2.0).to(t)
        s["qkv"] = x
        if case["packed"]:
            s["q"], s["k"] = x[:, :h], x[:, h : h + kv]
        else:
            s["q"], s["k"] = x[:, :h].contiguous(), x[:, h:].contiguous()
        for n in ("q", "k"):
            s[n + "_gamma"] = None if case["norm"] == "none" else 1.0 + _randn(g, d, std=0.1)
            s[n + "_beta"] = _randn(g, d, std=0.1) if case["norm"] == "layer" else None
            s[n + "_out"] = torch.empty(rows, h if n == "q" else kv, d, dtype=t, device=DEV)
        pos = torch.arange(case["table"], device=DEV, dtype=torch.float64)[:, None]
        ang = pos * 10000.0 ** (-torch.arange(r // 2, device=DEV, dtype=torch.float64) / (r // 2))
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        s["positions"] = torch.randint(case["table"], (rows,), device=DEV, generator=g) if case["given"] else None
        s["q_scale"] = math.log2(math.e) / math.sqrt(d)
    return s


# ---- the plain form ----


def _f32(x):
    return x.float()


def _fma(a, b, c):
    """a * b + c rounded to float32 once, as a fused multiply-add rounds it: the float64 product of float32 values is exact."""
    return _f32(a.double() * b.double() + c.double())


def _row_sum(cols, width):
    """The row sums of a running sum `cols(k, acc)` over columns, in float32 and in a stated order: 64 partial sums a row,
    partial 16 (b mod 4) + c over the 8 columns 8 c .. 8 c + 7 of the 128-column blocks b in ascending order; then folded in
    halves."""
    blocks = width // 128
    acc = None
    for b in range(0, blocks, 4):
        for e in range(8):
            acc = cols(b, e, acc)
    while acc.size(1) > 1:
        n = acc.size(1) // 2
        acc = acc[:, :n] + acc[:, n:]
    return acc


def _lanes(x):
    """[T, C] -> [T, blocks of 128 rounded up to a multiple of 4, 16, 8], zeros past the row."""
    t, c = x.shape
    pad = -c % 512
    return torch.nn.functional.pad(x, (0, pad)).view(t, -1, 16, 8)


def _normed(x, real, norm, gamma, beta, eps):
    """The norm of the first `real` columns, every step one float32 operation (fused multiply-adds where _fma stands)."""
    t, c = x.shape
    mask = torch.arange(c, device=x.device) < real
    if norm == "layer":
        xl = _lanes(torch.where(mask, x, torch.zeros_like(x)))
        s = _row_sum(lambda b, e, a: (lambda v: v if a is None else a + v)(xl[:, b : b + 4, :, e].reshape(t, 64)), c)
        mean = _f32(s.double() / real)
        d = torch.where(mask, x - mean, torch.zeros_like(x))
    else:
        d = torch.where(mask, x, torch.zeros_like(x))
    dl = _lanes(d)

    def square(b, e, a):
        v = dl[:, b : b + 4, :, e].reshape(t, 64)
        return v * v if a is None else _fma(v, v, a)

    var = _f32(_row_sum(square, c).double() / real)
    root = _f32((var + eps).double().sqrt())
    rstd = _f32(1.0 / root.double())
    d = d * rstd
    return _fma(d, gamma, beta) if norm == "layer" else d * gamma


def _rotated(v):
    """v blockdiag(H128): butterflies over column bits 0 to 6 in ascending order, each sum one float32 operation."""
    t, c = v.shape
    half = 1
    while half < 128:
        v = v.reshape(t, c // (2 * half), 2, half)
        v = torch.stack((v[:, :, 0] + v[:, :, 1], v[:, :, 0] - v[:, :, 1]), 2)
        half *= 2
    return v.reshape(t, c) * torch.tensor(ROOT128, dtype=torch.float32, device=v.device)


def _unit(e):
    """E8M0 exponents -> float32 powers of two, by their bits: 2^-127 is a subnormal number, 255 not a number."""
    bits = torch.where(e == 0, torch.full_like(e, 1 << 22), torch.where(e == 255, torch.full_like(e, 0x7FC00000), e << 23))
    return bits.to(torch.int32).view(torch.float32)


def _encode(v):
    """float32 [T, C] -> E2M1 magnitude codes and signs [T, C], and E8M0 exponents [T, C / 32] (255: not finite)."""
    t, c = v.shape
    blocks = v.reshape(t, c // 32, 32)
    amax = blocks.abs().amax(-1)
    finite = torch.isfinite(amax)
    e = (torch.frexp(torch.where(finite, amax, torch.ones_like(amax)))[1] - 3).clamp(min=-127)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    u = blocks.abs().double() * ((1023 - e.long()) << 52).view(torch.float64)[..., None]
    u = torch.where(finite[..., None], u, torch.zeros_like(u))
    # spacing 1/2 below 2, 1 below 4, 2 above; torch.round takes ties to even, which is E2M1's even code
    mag = torch.where(u < 2, torch.round(u * 2), torch.where(u < 4, torch.round(u) + 2, torch.round(u / 2) + 4)).clamp(max=7)
    biased = torch.where(finite, e + 127, torch.full_like(e, 255))
    return mag.long().reshape(t, c), (v < 0).long(), biased


def _decode(codes, scale):
    """MX4 -> float32 values [T, C]."""
    t, c = codes.size(0), codes.size(1) * 2
    nib = torch.stack((codes & 15, codes >> 4), -1).reshape(t, c // 32, 32).long()
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)
    word = torch.stack([(scale >> (8 * i)) & 255 for i in range(4)], -1).permute(1, 0, 2).reshape(t, c // 32)
    return (grid[nib] * _unit(word)[..., None]).reshape(t, c)


def _plain_quant(s):
    x = _f32(s["x"])
    if s["norm"] != "none":
        x = _normed(x, s["real"], s["norm"], s["gamma"], s["beta"], 1e-6)
    if s["rotate"]:
        x = _rotated(x)
    mag, sign, e = _encode(x)
    grid = torch.tensor(GRID, device=x.device)
    v = (grid[mag] * (1 - 2 * sign)).view(x.size(0), -1, 32) * _unit(e)[..., None]
    return v.reshape(x.shape).to(s["x"].dtype)


def _plain_gemm(s):
    y = _decode(s["a"], s["a_scale"]) @ _decode(s["w"], s["w_scale"]).t() + s["bias"]
    if s["epi"] == "residual":
        y = y + _f32(s["residual"])
    elif s["epi"] == "gelu":
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y**3)))
    elif s["epi"] == "swiglu":
        gate = y[:, 0::2]
        y = gate / (1.0 + torch.exp(-gate)) * y[:, 1::2]
    return y.to(s["out"].dtype)


def _plain_head(x, gamma, beta, norm, cos, sin, pairs, factor):
    t = x.dtype
    x = _f32(x)
    if norm == "layer":
        x = x - x.mean(-1, keepdim=True)
    if norm != "none":
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gamma
    if norm == "layer":
        x = x + beta
    r = 2 * cos.size(-1)
    cos, sin = cos[:, None], sin[:, None]
    if pairs:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., : r // 2], x[..., r // 2 : r]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return (torch.cat((turned, x[..., r:]), -1) * factor).to(t)


def _plain_qk(s):
    pos = s["positions"] if s["given"] else torch.arange(s["rows"], device=DEV) % s["table"]
    cos, sin = s["cos"][pos], s["sin"][pos]
    return (_plain_head(s["q"], s["q_gamma"], s["q_beta"], s["norm"], cos, sin, s["pairs"], s["q_scale"]),
            _plain_head(s["k"], s["k_gamma"], s["k_beta"], s["norm"], cos, sin, s["pairs"], 1.0))


# ---- one pass ----


def run(s):
    if not own:
        return {"quant": _plain_quant, "gemm": _plain_gemm, "qk": _plain_qk}[s["kind"]](s)
    from foidfinder_amd import kernels as ops

    norms = {"none": ops.NORM_NONE, "rms": ops.NORM_RMS, "layer": ops.NORM_LAYER}
    if s["kind"] == "quant":
        ops.quant_mx4(s["x"], s["codes"], s["scale"], s["rotate"], norms[s["norm"]], s["gamma"], s["beta"], s["real"], 1e-6)
        ops.dequant_mx4(s["codes"], s["scale"], s["out"])
        return s["out"]
    if s["kind"] == "gemm":
        epi = {"bias": ops.EPI_BIAS_F16, "residual": ops.EPI_RESIDUAL, "gelu": ops.EPI_GELU_F16, "swiglu": ops.EPI_SWIGLU}[s["epi"]]
        ops.gemm_mx4(s["a"], s["a_scale"], s["w"], s["w_scale"], s["bias"], s["out"], epi, 0, s["residual"])
        return s["out"]
    ops.qk_norm_rope(s["q"], s["k"], s["q_out"], s["k_out"], norms[s["norm"]], s["q_gamma"], s["k_gamma"], s["q_beta"],
                     s["k_beta"], s["cos"], s["sin"], s["positions"], s["pairs"], 1e-6, s["q_scale"])
    return s["q_out"], s["k_out"]


def work(case):
    rows, size = case["rows"], {"fp16": 2, "bf16": 2, "fp32": 4}[case["type"]]
    if case["kind"] == "quant":
        w = case["width"]
        rotation = 8 if case["rotate"] else 0  # seven butterfly stages and the factor
        norm = {"none": 0, "rms": 4, "layer": 7}[case["norm"]]
        return {"bytes": 2 * size * rows * w, "flops": rows * w * (rotation + norm + 3)}
    if case["kind"] == "gemm":
        n, k = case["cols"], case["width"]
        out = rows * (n // 2 if case["epi"] == "swiglu" else n) * size
        extra = rows * n * size if case["epi"] == "residual" else 0
        return {"bytes": (rows + n) * (k // 2 + k // 32) + 4 * n + out + extra, "flops": 2 * rows * n * k}
    heads, d = case["heads"] + case["kv"], case["dim"]
    entries = min(rows, case["table"]) * case["rot"] * 4
    return {"bytes": 2 * size * rows * heads * d + entries + (8 * rows if case["given"] else 0), "flops": 10 * rows * heads * d}


# ---- the operators' definitions in 64 bits ----


def _hadamard128():
    i = torch.arange(128, device=DEV)
    bits = i[:, None] & i[None]
    parity = sum((bits >> n) & 1 for n in range(7)) % 2
    return (1.0 - 2.0 * parity.double()) / math.sqrt(128.0)


def _values64(codes, scale):
    rows, width = codes.size(0), 2 * codes.size(1)
    out = torch.empty(rows, width, dtype=torch.float64, device=codes.device)
    for half, nib in ((0, codes & 15), (1, codes >> 4)):
        n = nib.double()
        low = n % 8
        mag = torch.where(low < 2, low / 2, (1 + (low % 2) / 2) * 2.0 ** (torch.floor(low / 2) - 1))
        out[:, half::2] = torch.where(n >= 8, -mag, mag)
    for i in range(width // 32):
        e = (scale[i // 4].long() >> (8 * (i % 4))) & 255
        f = torch.where(e == 255, math.nan, 2.0 ** (e.double() - 127.0))
        out[:, 32 * i : 32 * i + 32] *= f[:, None]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quant":
        real, outs = case["real"], []
        for x in s["x"].split(max(1, (1 << 24) // case["width"])):
            v = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
            v[:, :real] = x[:, :real].double()
            if case["norm"] == "none":
                v = x.double()
            else:
                h = v[:, :real]
                if case["norm"] == "layer":
                    h = h - h.mean(1, keepdim=True)
                h = h * (h.square().mean(1, keepdim=True) + 1e-6).rsqrt() * s["gamma"][:real].double()
                v[:, :real] = h + s["beta"][:real].double() if case["norm"] == "layer" else h
            if case["rotate"]:
                v = (v.view(-1, 128) @ _hadamard128()).view(v.shape)
            v = v.view(-1, 32)
            top = v.abs().amax(1, keepdim=True)
            unit = ((torch.frexp(top)[1].long() - 3).clamp(min=-127) + 1023 << 52).view(torch.float64)
            u = v / unit
            # nearest of the 15 values; at a midpoint the one with the even code
            mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=DEV)
            up = torch.tensor([False, True, False, True, False, True, False], device=DEV)
            m = u.abs()
            code = sum(((m > b) | ((m == b) & t)).long() for b, t in zip(mids, up))
            grid = torch.tensor(GRID, dtype=torch.float64, device=DEV)
            outs.append((torch.sign(u) * grid[code] * unit).view(x.shape))
        return torch.cat(outs)
    if case["kind"] == "gemm":
        y = _values64(s["a"], s["a_scale"]) @ _values64(s["w"], s["w_scale"]).t()
        y += s["bias"].double()
        if case["epi"] == "residual":
            y += s["residual"].double()
        elif case["epi"] == "gelu":
            y = y / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
        elif case["epi"] == "swiglu":
            p = y.view(y.size(0), -1, 2)
            y = torch.sigmoid(p[..., 0]) * p[..., 0] * p[..., 1]
        return y
    row = torch.arange(case["rows"], device=DEV) % case["table"] if s["positions"] is None else s["positions"]
    turn = torch.complex(s["cos"].double(), s["sin"].double())[row].unsqueeze(1)
    outs = []
    for n, factor in (("q", s["q_scale"]), ("k", 1.0)):
        x = s[n].double()
        if case["norm"] == "layer":
            x = (x - x.mean(-1, keepdim=True)) * (x.var(-1, keepdim=True, unbiased=False) + 1e-6).rsqrt()
            x = x * s[n + "_gamma"].double() + s[n + "_beta"].double()
        elif case["norm"] == "rms":
            x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * s[n + "_gamma"].double()
        head, tail = x[..., : case["rot"]], x[..., case["rot"] :]
        if case["pairs"]:
            z = torch.view_as_complex(head.reshape(*head.shape[:-1], -1, 2).contiguous()) * turn
            head = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(*head.chunk(2, -1)) * turn
            head = torch.cat((z.real, z.imag), -1)
        outs.append(torch.cat((head, tail), -1) * factor)
    return tuple(outs)
