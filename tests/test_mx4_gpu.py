"""MX4 quantization and product and the head norm on the GPU, against the oracles.

Bars: codes and exponents equal to the oracle's (zeros of either sign are one value); dequantized values exact; products
within the rounding of an fp32 summation plus half a step of the output, and exactly equal where every partial sum is
representable; the head norm within fp32 rounding of its terms plus half a step of the output.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import attention as OA
from oracle import gemm as OG
from oracle import mx4 as OX
from oracle import qk_norm as OQ

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
HALF = {"fp16": 2.0**-11, "bf16": 2.0**-8, "fp32": 2.0**-24}  # half a step, relative
TINY = {"fp16": 2.0**-25, "bf16": 2.0**-126, "fp32": 2.0**-126}  # half a step of the smallest numbers (subnormal for fp16)


def kern():
    from foidfinder_amd import kernels as K

    return K


def gpu(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def typed(a, kind, dev):
    """A float32 array as a tensor of the type on the GPU, and its values back in float32."""
    t = gpu(a.astype(np.float32), dev).to(TYPES[kind])
    return t, t.float().cpu().numpy()


def empty_mx4(T, C, dev):
    """Outputs between guard bytes: (codes, scale, check) where check() says whether the guards are as they were."""
    buf = torch.full((T * C // 2 + 512,), 0x5A, dtype=torch.uint8, device=dev)
    words = torch.full((C // 128 * T + 64,), 0x5A5A5A5A, dtype=torch.int32, device=dev)

    def check():
        b, w = buf.cpu().numpy(), words.cpu().numpy()
        return (b[:256] == 0x5A).all() and (b[-256:] == 0x5A).all() and (w[:32] == 0x5A5A5A5A).all() \
            and (w[-32:] == 0x5A5A5A5A).all()

    return buf[256:-256].view(T, C // 2), words[32:-32].view(C // 128, T), check


def assert_same_mx4(got, want):
    (gc, ge), (wc, we) = OX.unpack(*(t.cpu().numpy() for t in got)), OX.unpack(*want)
    bad = np.argwhere(ge != we)
    assert bad.size == 0, f"{len(bad)} exponents differ, first {bad[:4].tolist()}: {ge[tuple(bad[0])]} vs {we[tuple(bad[0])]}"
    live = np.repeat(we != 255, 32, axis=1)
    gc, wc = (np.where(c == 8, 0, c) for c in (gc, wc))  # -0 is 0
    bad = np.argwhere((gc != wc) & live)
    assert bad.size == 0, f"{len(bad)} codes differ, first {bad[:4].tolist()}: {gc[tuple(bad[0])]} vs {wc[tuple(bad[0])]}"


def activations(rng, T, C):
    x = rng.standard_normal((T, C)).astype(np.float32)
    x[:, rng.choice(C, max(1, C // 100), replace=False)] *= 20.0
    return x


def run_quant(dev, x, kind, rotate, norm, c_real=0, gamma=None, beta=None, eps=1e-6):
    t, back = typed(x, kind, dev)
    codes, scale, check = empty_mx4(*x.shape, dev)
    g, b = (None if p is None else gpu(p, dev) for p in (gamma, beta))
    kern().quant_mx4(t, codes, scale, rotate, norm, g, b, c_real, eps)
    torch.cuda.synchronize()
    assert check(), "wrote outside its outputs"
    want = OX.quant_mx4(back, rotate, norm, c_real, gamma, beta, eps)
    return (codes, scale), want


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("rotate", [True, False])
@pytest.mark.parametrize(("T", "C"), [(1, 128), (1, 4736), (5, 512), (3, 640), (70, 768), (1025, 1024), (9, 6144)])
def test_quant_mx4_bit_exact(dev, rng, T, C, rotate, kind):
    assert_same_mx4(*run_quant(dev, activations(rng, T, C), kind, rotate, OX.NONE))


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("norm", [OX.RMS, OX.LAYER])
@pytest.mark.parametrize(("T", "C", "c_real", "rotate"), [(1, 128, 1, True), (1, 128, 128, False), (7, 256, 130, True),
                                                          (70, 768, 768, True), (1025, 1024, 1024, True),
                                                          (33, 1024, 1000, False), (130, 2816, 2730, True),
                                                          (2, 4736, 4736, True), (5, 6144, 6100, True),
                                                          (3, 1408, 1280, True), (3, 640, 5, True)])
def test_quant_mx4_norm_bit_exact(dev, rng, T, C, c_real, rotate, norm, kind):
    """Padding columns hold values that must not count, one of them infinite."""
    x = activations(rng, T, C)
    if c_real < C:
        x[:, C - 1] = np.inf
    g, b = np.zeros(C, np.float32), np.zeros(C, np.float32)
    g[:c_real] = 1 + 0.1 * rng.standard_normal(c_real)
    b[:c_real] = 0.1 * rng.standard_normal(c_real)
    assert_same_mx4(*run_quant(dev, x, kind, rotate, norm, c_real, g, b if norm == OX.LAYER else None))


@pytest.mark.parametrize("rotate", [True, False])
def test_quant_mx4_special_rows(dev, rotate):
    x = np.zeros((10, 256), np.float32)
    x[1, 0], x[2, 255] = 1.0, -3.5
    x[3] = 0.25
    x[4, ::3], x[4, 1::3] = 3e38, -3e38  # the rotation's sums overflow
    x[5, 40], x[6, 200] = np.inf, np.nan
    x[7] = 2.0**-133  # subnormal in bf16: the exponent stops at -127
    x[8] = np.tile(np.arange(-16, 16) * 0.25, 8)  # every midpoint of the grid, 8 ties' neighbours included
    x[8, 31::32] = 7.75
    x[9] = np.where(np.arange(256) % 2, 6.0, -7.0)
    got, want = run_quant(dev, x, "bf16", rotate, OX.NONE)
    assert_same_mx4(got, want)
    e = OX.unpack(*want)[1]
    assert (e[5, :4] == 255).any() and (e[5, 4:] != 255).all() and (e[6, 4:] == 255).any()
    x16 = x.copy()
    x16[4] = np.where(x[4] == 0, 0, np.sign(x[4]) * 65504)
    assert_same_mx4(*run_quant(dev, x16, "fp16", rotate, OX.NONE))


@pytest.mark.parametrize("norm", [OX.RMS, OX.LAYER])
@pytest.mark.parametrize(("T", "C"), [(6, 640), (6, 1024), (4100, 640), (4100, 768)])
def test_quant_mx4_norm_special_rows(dev, rng, T, C, norm):
    """A row that holds a NaN has no codes (every exponent 255), one with an infinity those of the formula; the rows beside
    them, some in the same wave, are as without them. Rows of zeros and of one value."""
    x = activations(rng, T, C)
    x[0, 3], x[2, C - 1], x[3] = np.inf, np.nan, 0
    x[4] = 0.5
    g, b = np.ones(C, np.float32), np.linspace(-1, 1, C).astype(np.float32)
    got, want = run_quant(dev, x, "bf16", True, norm, C, g, b if norm == OX.LAYER else None)
    assert_same_mx4(got, want)
    e = OX.unpack(*(t.cpu().numpy() for t in got))[1]
    assert (e[2] == 255).all() and (e[[1, 3, 4, 5]] != 255).all()


@pytest.mark.parametrize("norm", [OX.NONE, OX.LAYER])
def test_quant_mx4_strided_rows(dev, rng, norm):
    x = rng.standard_normal((6, 1040)).astype(np.float32)
    t = gpu(x.astype(np.float16), dev)[:, 8:776]
    codes, scale, check = empty_mx4(6, 768, dev)
    g, b = (np.ones(768, np.float32), np.zeros(768, np.float32)) if norm else (None, None)
    kern().quant_mx4(t, codes, scale, True, norm, *(None if p is None else gpu(p, dev) for p in (g, b)))
    want = OX.quant_mx4(x.astype(np.float16).astype(np.float32)[:, 8:776], True, norm, 0, g, b)
    assert check()
    assert_same_mx4((codes, scale), want)
    # an expanded row: every row the same memory is refused (it lies closer than C)
    with pytest.raises(RuntimeError, match="x_stride"):
        kern().quant_mx4(t[:1].expand(6, 768), codes, scale)


@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp32"])
def test_dequant_mx4_exact(dev, rng, kind):
    code = np.concatenate([np.tile(np.arange(16, dtype=np.uint8), (4, 16)),
                           rng.integers(0, 16, (33, 256)).astype(np.uint8)])
    e = rng.integers(100, 150, (37, 8)).astype(np.uint8)
    e[0], e[1, :4], e[2] = 255, 0, [0, 1, 2, 3, 251, 252, 253, 254]
    packed = OX.pack(code, e)
    out = torch.zeros(37, 256, dtype=TYPES[kind], device=dev)
    kern().dequant_mx4(gpu(packed[0], dev), gpu(packed[1], dev), out)
    want64 = OX.values(*packed)
    with np.errstate(over="ignore"):
        want = torch.from_numpy(want64.astype(np.float32)).to(TYPES[kind])  # float32 holds every value but 6 * 2^127
    got, want = out.cpu().double().numpy(), want.double().numpy()
    assert np.array_equal(got, want, equal_nan=True)


# ---- product ----

VARIANTS = [0, 1, 2, 3, 4, 5]
SHAPES = [(1, 1, 128), (1, 2304, 768), (3, 17, 256), (16, 1000, 1152), (33, 31, 384), (64, 66, 128), (130, 257, 640),
          (300, 1024, 2816), (257, 514, 1024), (1025, 768, 1024)]


def test_gemm_mx4_variant_list_is_complete(dev):
    assert kern().lib().ff_gemm_mx4_variants() == max(VARIANTS)


def random_mx4(rng, T, C, lo, hi):
    return OX.pack(rng.integers(0, 16, (T, C)).astype(np.uint8), rng.integers(lo, hi, (T, C // 32)).astype(np.uint8))


def run_gemm(dev, a, w, bias, kind, epi, variant, residual=None):
    """The product into memory between guard rows."""
    M, N = a[0].shape[0], w[0].shape[0]
    cols = N // 2 if epi == OG.EPI_SWIGLU else N
    pad = 64
    buf = torch.full((M * cols + 2 * pad,), 7.0, dtype=TYPES[kind], device=dev)
    out = buf[pad : pad + M * cols].view(M, cols)
    ts = [gpu(t, dev) for t in (*a, *w)]
    kern().gemm_mx4(*ts, None if bias is None else gpu(bias, dev), out, epi, variant,
                    None if residual is None else residual)
    torch.cuda.synchronize()
    assert (buf[:pad] == 7).all() and (buf[pad + M * cols :] == 7).all(), "wrote outside its output"
    return out.double().cpu().numpy()


def sum_error(K, size):
    """Rounding of an fp32 sum of K exact products and a bias in any order, each addition off by at most a whole step
    (2^-23, which also covers a truncating adder)."""
    return (K + 2) * 2.0**-23 * size


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize(("M", "N", "K"), SHAPES)
def test_gemm_mx4_exact_sums(dev, rng, M, N, K, variant):
    """Exponents of -1 .. 0 on both sides: every partial sum is a multiple of 2^-4 below 36 K < 2^17, so 21 bits hold it and
    any order of additions gives the exact sum. A wrong exponent, column or row shows as a wrong number."""
    a, w = random_mx4(rng, M, K, 126, 128), random_mx4(rng, N, K, 126, 128)
    got = run_gemm(dev, a, w, None, "fp32", OG.EPI_BIAS_F16, variant)
    want, _ = OX.gemm_mx4(a, w)
    bad = np.argwhere(got != want)
    assert bad.size == 0, f"{len(bad)} differ, first {bad[:4].tolist()}: {got[tuple(bad[0])]} vs {want[tuple(bad[0])]}"


def epilogue64(y, epi, residual):
    if epi == OG.EPI_RESIDUAL:
        return y + residual
    if epi == OG.EPI_GELU_F16:
        return y / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (y + 0.044715 * y**3)))
    if epi == OG.EPI_SWIGLU:
        g, v = y[:, 0::2], y[:, 1::2]
        return g / (1 + np.exp(-g)) * v
    return y


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("epi", [OG.EPI_BIAS_F16, OG.EPI_RESIDUAL, OG.EPI_GELU_F16, OG.EPI_SWIGLU])
@pytest.mark.parametrize(("M", "N", "K"), [(1, 2, 128), (5, 30, 384), (77, 130, 256), (513, 1024, 1152), (300, 776, 640)])
def test_gemm_mx4_epilogues(dev, rng, M, N, K, epi, kind, variant):
    """GELU's and SiLU's derivatives are below 1.13; their hardware exponential and reciprocal and the few products around
    them cost at most 16 fp32 steps of the result, and of the input's share (the exponent -2u carries u's relative
    rounding): 2^-19 (|y| + |result|) covers both."""
    a, w = random_mx4(rng, M, K, 120, 126), random_mx4(rng, N, K, 119, 125)
    bias = rng.standard_normal(N).astype(np.float32)
    res = typed(rng.standard_normal((M, N)), kind, dev) if epi == OG.EPI_RESIDUAL else (None, None)
    got = run_gemm(dev, a, w, bias, kind, epi, variant, res[0])
    y, size = OX.gemm_mx4(a, w, bias)
    want = epilogue64(y, epi, res[1])
    e = sum_error(K, size)
    if epi == OG.EPI_RESIDUAL:
        e = e + 2.0**-23 * np.abs(want)
    elif epi == OG.EPI_GELU_F16:
        e = 1.13 * e + 2.0**-19 * (np.abs(y) + np.abs(want))
    elif epi == OG.EPI_SWIGLU:
        g, v = y[:, 0::2], y[:, 1::2]
        e = (1.13 * e[:, 0::2] + 2.0**-19 * np.abs(g)) * (np.abs(v) + e[:, 1::2]) + np.abs(g) * e[:, 1::2]
    tol = e + HALF[kind] * (np.abs(want) + e) + TINY[kind]
    bad = np.argwhere(~(np.abs(got - want) <= tol))
    assert bad.size == 0, f"{len(bad)} off, first {bad[:4].tolist()}: {got[tuple(bad[0])]} vs {want[tuple(bad[0])]}"


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("M", [70, 64, 20])
def test_gemm_mx4_wide_exponents_and_blocks_that_are_not_numbers(dev, rng, M, variant):
    """Exponents over 2^+-30, every block with its own: a row with a block of exponent 255 is not a number in all of its
    products, and no other row is; residual in place."""
    N, K = 90, 640
    a, w = random_mx4(rng, M, K, 97, 158), random_mx4(rng, N, K, 97, 158)
    y, size = OX.gemm_mx4(a, w)
    got = run_gemm(dev, a, w, None, "fp32", OG.EPI_BIAS_F16, variant)
    assert (np.abs(got - y) <= sum_error(K, size)).all()
    ac, ae = OX.unpack(*a)
    wc, we = OX.unpack(*w)
    ae[M - 1, 19], we[31, 3] = 255, 255
    got = run_gemm(dev, OX.pack(ac, ae), OX.pack(wc, we), None, "fp32", OG.EPI_BIAS_F16, variant)
    want = y.copy()
    want[M - 1], want[:, 31] = np.nan, np.nan
    assert np.array_equal(np.isnan(got), np.isnan(want))
    out, x = typed(rng.standard_normal((M, N)), "bf16", dev)
    kern().gemm_mx4(*(gpu(t, dev) for t in (*a, *w)), None, out, OG.EPI_RESIDUAL, variant)
    want, got = y + x, out.double().cpu().numpy()
    e = sum_error(K, size) + 2.0**-23 * np.abs(want)
    assert (np.abs(got - want) <= e + HALF["bf16"] * (np.abs(want) + e)).all()


@pytest.mark.parametrize("variant", [0, 1, 2])
@pytest.mark.parametrize(("M", "N", "K"), [(16, 70001, 384), (64, 66000, 128), (33, 5001, 1152), (1, 40000, 640),
                                           (32, 33, 3840)])
def test_gemm_mx4_few_rows_exact(dev, rng, M, N, K, variant):
    """Up to 64 rows and many columns, odd unit counts, rows that start off a 4-byte boundary; exact as above."""
    a, w = random_mx4(rng, M, K, 126, 128), random_mx4(rng, N, K, 126, 128)
    bias = rng.integers(-8, 8, N).astype(np.float32)
    got = run_gemm(dev, a, w, bias, "fp32", OG.EPI_BIAS_F16, variant)
    av, wv = (torch.from_numpy(OX.values(*t).astype(np.float32)) for t in (a, w))
    want = (av @ wv.T).double().numpy() + bias  # float32 holds every partial sum, so torch's order does not matter
    bad = np.argwhere(got != want)
    assert bad.size == 0, f"{len(bad)} differ, first {bad[:4].tolist()}: {got[tuple(bad[0])]} vs {want[tuple(bad[0])]}"


def test_gemm_mx4_repeats_bit_for_bit(dev, rng):
    for M, N, K in ((1, 300, 1024), (200, 300, 640), (1500, 1100, 256)):
        a, w = random_mx4(rng, M, K, 118, 130), random_mx4(rng, N, K, 118, 130)
        first = run_gemm(dev, a, w, None, "fp32", OG.EPI_BIAS_F16, 0)
        assert np.array_equal(first, run_gemm(dev, a, w, None, "fp32", OG.EPI_BIAS_F16, 0))


def test_gemm_mx4_no_rows(dev):
    K = kern()
    e = torch.empty(0, 64, dtype=torch.uint8, device=dev), torch.empty(1, 0, dtype=torch.int32, device=dev)
    w = torch.zeros(8, 64, dtype=torch.uint8, device=dev), torch.zeros(1, 8, dtype=torch.int32, device=dev)
    K.gemm_mx4(*e, *w, None, torch.empty(0, 8, device=dev), K.EPI_BIAS_F16)
    K.quant_mx4(torch.empty(0, 128, dtype=torch.half, device=dev), *e)
    K.dequant_mx4(*e, torch.empty(0, 128, device=dev))
    q, ko = (torch.empty(0, n, 64, dtype=torch.half, device=dev) for n in (4, 2))
    t = torch.ones(3, 32, device=dev)
    K.qk_norm_rope(q, ko, q, ko, K.NORM_NONE, None, None, None, None, t, t)
    K.qk_norm_rope(q, ko, q, ko, K.NORM_NONE, None, None, None, None, t, t, torch.empty(0, dtype=torch.int32, device=dev))


@pytest.mark.parametrize("variant", VARIANTS)
def test_gemm_mx4_offsets_past_32_bits(dev, rng, variant):
    """An output of 2.3 G elements (4.6 GB): rows whose offsets pass 2^31 elements, the sums exact as above and rounded
    once to bf16."""
    K = kern()
    M, N, Kd = 70001, 32770, 128
    w = random_mx4(rng, N, Kd, 126, 128)
    few = random_mx4(rng, 5, Kd, 126, 128)
    rows = np.array([0, 65536, 65537, 70000, 33000])
    codes = torch.zeros(M, Kd // 2, dtype=torch.uint8, device=dev)
    scale = torch.zeros(1, M, dtype=torch.int32, device=dev)
    codes[rows] = gpu(few[0], dev)
    scale[:, rows] = gpu(few[1], dev)
    out = torch.empty(M, N, dtype=torch.bfloat16, device=dev)
    K.gemm_mx4(codes, scale, *(gpu(t, dev) for t in w), None, out, K.EPI_BIAS_F16, variant)
    want = torch.from_numpy(OX.gemm_mx4(few, w)[0]).to(torch.bfloat16)
    assert torch.equal(out[rows].cpu(), want)
    assert not out[1].any() and not out[69999].any()


@pytest.mark.parametrize("norm", [OX.NONE, OX.RMS])
def test_quant_mx4_offsets_past_32_bits(dev, rng, norm):
    """2.2 G elements: the last rows start past 2^31 elements of x and 2^30 bytes of codes."""
    K = kern()
    T, C = 360_000, 6144
    x = torch.zeros(T, C, dtype=torch.half, device=dev)
    last, back = typed(activations(rng, 3, C), "fp16", dev)
    x[-3:] = last
    codes = torch.empty(T, C // 2, dtype=torch.uint8, device=dev)
    scale = torch.empty(C // 128, T, dtype=torch.int32, device=dev)
    g = np.ones(C, np.float32) if norm else None
    K.quant_mx4(x, codes, scale, True, norm, None if g is None else gpu(g, dev))
    assert_same_mx4((codes[-3:], scale[:, -3:]), OX.quant_mx4(back, True, norm, 0, g))
    assert not scale[:, :-3].any() and not (codes[:-3] & 0x77).any()  # zeros: the lowest exponent, either sign
    x.fill_(7.0)
    K.dequant_mx4(codes, scale, x)
    want = OX.values(codes[-3:].cpu().numpy(), scale[:, -3:].cpu().numpy())
    assert np.array_equal(x[-3:].double().cpu().numpy(), want) and not x[:-3].any()


def test_mx4_ops_refuse_tensors_that_autograd_follows(dev):
    """Through the dispatcher as well, where no autograd kernel stands before the op."""
    K = kern()
    x = torch.zeros(2, 128, dtype=torch.half, device=dev, requires_grad=True)
    codes, scale, _ = empty_mx4(2, 128, dev)
    for op in (K.quant_mx4, K.kernels().quant_mx4):
        with pytest.raises(RuntimeError, match="backward"):
            op(x, codes, scale)
        with torch.no_grad():
            op(x, codes, scale)


# ---- head norm and rotation ----


def tables(rng, L, R):
    ang = rng.uniform(-np.pi, np.pi, (L, R // 2))
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def check_qk(got, x, norm, gamma, beta, cos, sin, pos, pairs, scale, kind):
    """Half a step of the output, and fp32's share: the norm's mean, variance, quotient and products cost under 24 half
    steps relative to a value's own terms, the rotation's two products and sum and the scale 4 more; a mean over D columns
    of values up to 8 deviations adds D / 8 half steps of the normed size. 2^-17 of the terms, and of one (the normed size)
    for the LayerNorm's difference, covers them."""
    want, size = OQ.qk_norm_rope(x, norm, gamma, beta, 1e-6, cos, sin, pos, pairs, scale)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    got, want = np.nan_to_num(got), np.nan_to_num(want)
    e = 2.0**-17 * (size + (abs(scale) if norm == OQ.LAYER else 0))
    tol = e + HALF[kind] * (np.abs(want) + e) + TINY[kind]
    bad = np.argwhere(~(np.abs(got - want) <= tol))
    assert bad.size == 0, f"{len(bad)} off, first {bad[:4].tolist()}: {got[tuple(bad[0])]} vs {want[tuple(bad[0])]}"


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("norm", [OQ.NONE, OQ.RMS, OQ.LAYER])
@pytest.mark.parametrize("pairs", [True, False])
@pytest.mark.parametrize(("T", "H", "KV", "D", "R", "L"), [
    (1, 1, 1, 8, 8, 1), (1, 32, 8, 128, 128, 50), (5, 3, 1, 64, 64, 2), (33, 16, 16, 64, 64, 33), (7, 4, 2, 80, 80, 9),
    (6, 5, 5, 96, 24, 6), (9, 2, 2, 256, 256, 11), (4, 8, 4, 256, 72, 7), (130, 6, 2, 128, 64, 17), (3, 2, 1, 40, 16, 5),
    (1027, 3, 3, 64, 48, 1025), (2, 70, 30, 128, 128, 3), (5, 3, 2, 96, 32, 4), (9, 2, 1, 48, 16, 9), (6, 3, 2, 192, 176, 5),
    (3, 2, 2, 240, 240, 3)])
def test_qk_norm_rope(dev, rng, T, H, KV, D, R, L, pairs, norm, kind):
    """Packed rows: q and k are views of [T, H + 2 KV, D], and the packed outputs' value columns stay as they were."""
    K = kern()
    qkv, back = typed(2 * rng.standard_normal((T, H + 2 * KV, D)) + 0.3, kind, dev)
    cos, sin = tables(rng, L, R)
    g = [(1 + 0.1 * rng.standard_normal(D)).astype(np.float32) if norm else None for _ in range(2)]
    b = [(0.1 * rng.standard_normal(D)).astype(np.float32) if norm == OQ.LAYER else None for _ in range(2)]
    out = torch.full_like(qkv, 7.0)
    up = lambda a: None if a is None else gpu(a, dev)  # noqa: E731
    args = (norm, up(g[0]), up(g[1]), up(b[0]), up(b[1]), gpu(cos, dev), gpu(sin, dev))
    K.qk_norm_rope(qkv[:, :H], qkv[:, H : H + KV], out[:, :H], out[:, H : H + KV], *args, None, pairs, 1e-6, 0.37)
    got = out.double().cpu().numpy()
    assert (got[:, H + KV :] == 7).all()
    pos = np.arange(T) % L
    check_qk(got[:, :H], back[:, :H], norm, g[0], b[0], cos, sin, pos, pairs, 0.37, kind)
    check_qk(got[:, H : H + KV], back[:, H : H + KV], norm, g[1], b[1], cos, sin, pos, pairs, 1.0, kind)
    # in place: the same values, v untouched
    inplace = qkv.clone()
    K.qk_norm_rope(inplace[:, :H], inplace[:, H : H + KV], inplace[:, :H], inplace[:, H : H + KV], *args, None, pairs, 1e-6,
                   0.37)
    assert torch.equal(inplace[:, : H + KV], out[:, : H + KV]) and torch.equal(inplace[:, H + KV :], qkv[:, H + KV :])


@pytest.mark.parametrize("int_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("pairs", [True, False])
def test_qk_norm_rope_positions_and_layouts(dev, rng, pairs, int_type):
    """Positions in any order, twice the same, outside the table on both sides (also far outside, past 32 bits where the type
    holds it); outputs with the heads outermost, inputs that share one row over the heads, strides of 8 bytes only."""
    K = kern()
    T, H, KV, D, R, L = 9, 4, 2, 64, 32, 6
    cos, sin = tables(rng, L, R)
    far = 1 << 40 if int_type == torch.int64 else 2**31 - 1
    pos = np.array([5, 0, 0, 3, 6, -1, 2, far, -far - (int_type == torch.int32)])
    buf, back = typed(rng.standard_normal((T, H * D + 4)), "fp16", dev)
    q = buf[:, : H * D].unflatten(1, (H, D))
    k = buf[:, 4 : 4 + D].unsqueeze(1).expand(T, KV, D)
    g = [np.ones(D, np.float32), (1 + 0.1 * rng.standard_normal(D)).astype(np.float32)]
    qo = torch.empty(H, T, D, dtype=torch.half, device=dev).transpose(0, 1)
    ko = torch.full((KV, T + 3, D), 7.0, dtype=torch.half, device=dev)
    K.qk_norm_rope(q, k, qo, ko[:, 1 : T + 1].transpose(0, 1), OQ.RMS, gpu(g[0], dev), gpu(g[1], dev), None, None,
                   gpu(cos, dev), gpu(sin, dev), gpu(pos, dev).to(int_type), pairs)
    xq = back[:, : H * D].reshape(T, H, D)
    xk = np.repeat(back[:, None, 4 : 4 + D], KV, axis=1)
    check_qk(qo.double().cpu().numpy(), xq, OQ.RMS, g[0], None, cos, sin, pos, pairs, 1.0, "fp16")
    got = ko.double().cpu().numpy()
    check_qk(got[:, 1 : T + 1].transpose(1, 0, 2), xk, OQ.RMS, g[1], None, cos, sin, pos, pairs, 1.0, "fp16")
    assert (got[:, 0] == 7).all() and (got[:, T + 1 :] == 7).all()


@pytest.mark.parametrize("pairs", [True, False])
@pytest.mark.parametrize(("D", "R"), [(64, 64), (128, 96), (256, 16), (48, 32)])
def test_qk_norm_rope_is_the_same_at_any_alignment(dev, rng, D, R, pairs):
    """Rows from multiples of 16 bytes and of 8 only take different accesses and the same arithmetic."""
    K = kern()
    T, H = 37, 5
    x, _ = typed(rng.standard_normal((T, H, D)), "bf16", dev)
    cos, sin = (gpu(t, dev) for t in tables(rng, T, R))
    g = gpu((1 + 0.1 * rng.standard_normal(D)).astype(np.float32), dev)
    outs = []
    for shift in (0, 4):
        rows = torch.full((T, H * D + 8), 7.0, dtype=torch.bfloat16, device=dev)
        y = rows[:, shift : shift + H * D].unflatten(1, (H, D))
        o = torch.full_like(rows, 7.0)
        y.copy_(x)
        K.qk_norm_rope(y, x, o[:, shift : shift + H * D].unflatten(1, (H, D)), torch.empty_like(x), OQ.RMS, g, g, None, None,
                       cos, sin, None, pairs)
        assert (o[:, :shift] == 7).all() and (o[:, shift + H * D :] == 7).all()
        outs.append(o[:, shift : shift + H * D].clone())
    assert torch.equal(*outs)


def test_qk_norm_rope_offsets_past_32_bits(dev, rng):
    """A token stride of 600 M elements: the last token starts past 2^31 elements (4.8 GB) of q and of its output."""
    K = kern()
    D, step = 64, 600_000_000
    big = torch.empty(4 * step + 2 * D, dtype=torch.half, device=dev)
    q = big.as_strided((5, 1, D), (step, D, 1))
    qo = big.as_strided((5, 1, D), (step, D, 1), D)
    x, back = typed(rng.standard_normal((5, 1, D)), "fp16", dev)
    q.copy_(x)
    cos, sin = tables(rng, 5, D)
    g = np.ones(D, np.float32)
    ko = torch.empty_like(x)
    K.qk_norm_rope(q, x, qo, ko, OQ.RMS, gpu(g, dev), gpu(g, dev), None, None, gpu(cos, dev), gpu(sin, dev))
    check_qk(qo.double().cpu().numpy(), back, OQ.RMS, g, None, cos, sin, np.arange(5), True, 1.0, "fp16")
    assert torch.equal(qo.contiguous(), ko)


def test_qk_norm_rope_norms_of_zero_and_large_heads(dev):
    """Zeros stay zeros (eps keeps the quotient finite); fp16's largest values, whose squares fp16 cannot hold, are normed."""
    K = kern()
    x = torch.zeros(2, 2, 64, dtype=torch.half, device=dev)
    x[1] = 65504.0
    x[1, 1, ::2] = -65504.0
    g = torch.ones(64, device=dev)
    cos, sin = torch.ones(2, 32, device=dev), torch.zeros(2, 32, device=dev)
    o, o2 = torch.empty_like(x), torch.empty_like(x)
    K.qk_norm_rope(x, x, o, o2, OQ.RMS, g, g, None, None, cos, sin)
    assert not o[0].any() and torch.equal(o, o2)
    assert torch.equal(o[1], x[1].sign())


@pytest.mark.parametrize("norm", [OQ.NONE, OQ.RMS, OQ.LAYER])
def test_qk_norm_rope_keeps_values_that_are_not_finite_to_their_head(dev, rng, norm):
    """Columns past the rotated ones and heads beside the fault are as without it; the fault's head shows it."""
    K = kern()
    x, _ = typed(rng.standard_normal((5, 3, 80)), "bf16", dev)
    cos, sin = (gpu(t, dev) for t in tables(rng, 5, 32))
    g = torch.ones(80, device=dev) if norm else None
    b = torch.zeros(80, device=dev) if norm == OQ.LAYER else None
    outs = []
    for fault in (False, True):
        y = x.clone()
        if fault:
            y[1, 2, 7], y[3, 0, 79] = float("nan"), float("inf")
        o, o2 = torch.empty_like(y), torch.empty_like(y)
        K.qk_norm_rope(y, y, o, o2, norm, g, g, b, b, cos, sin)
        assert torch.equal(o.view(torch.int16), o2.view(torch.int16))
        outs.append(o)
    bad = torch.zeros(5, 3, dtype=torch.bool, device=dev)
    bad[1, 2] = bad[3, 0] = True
    assert torch.equal(outs[0][~bad], outs[1][~bad])
    assert outs[1][1, 2].isnan().any() and not outs[1][3, 0].isfinite().all()


# ---- together ----


def test_mx4_block_eager_and_captured(dev, rng):
    """The attention half of a block on these operators, as they are used together: norm + rotation + codes, the QKV product,
    head norms and rotation in place, attention, rotation + codes, the projection added to the stream; eagerly on a side
    stream, then captured and replayed with eager work in between. Each step is checked against its oracle from the previous
    step's own output, and every replay against the eager run bit for bit."""
    K = kern()
    L, seqs, H = 65, 3, 4
    C, T = H * 64, L * seqs
    x, back = typed(activations(rng, T, C), "fp16", dev)
    g, b = (1 + 0.1 * rng.standard_normal(C)).astype(np.float32), (0.1 * rng.standard_normal(C)).astype(np.float32)
    wq, wo = (rng.standard_normal((n, C)).astype(np.float32) / 16 for n in (3 * C, C))
    weights = []
    for w in (wq, wo):
        t = gpu(w.astype(np.float16), dev)
        codes, scale, _ = empty_mx4(w.shape[0], C, dev)
        K.quant_mx4(t, codes, scale)
        assert_same_mx4((codes, scale), OX.quant_mx4(w.astype(np.float16).astype(np.float32)))
        weights.append((codes, scale))
    bias = [rng.standard_normal(n).astype(np.float32) * 0.1 for n in (3 * C, C)]
    hg = [(1 + 0.1 * rng.standard_normal(64)).astype(np.float32) for _ in range(2)]
    cos, sin = tables(rng, L, 64)
    dg, db, dh, dc, ds = gpu(g, dev), gpu(b, dev), [gpu(t, dev) for t in hg], gpu(cos, dev), gpu(sin, dev)
    dbias = [gpu(t, dev) for t in bias]
    codes, scale, _ = empty_mx4(T, C, dev)
    codes2, scale2, _ = empty_mx4(T, C, dev)
    qkv, o, out = (torch.empty(T, n, dtype=torch.half, device=dev) for n in (3 * C, C, C))
    plain = torch.empty_like(qkv)
    ops, q_scale = K.kernels(), 0.125 * 1.4426950408889634

    def forward():
        ops.quant_mx4(x, codes, scale, True, K.NORM_LAYER, dg, db, 0, 1e-6)
        ops.gemm_mx4(codes, scale, *weights[0], dbias[0], qkv, K.EPI_BIAS_F16)
        plain.copy_(qkv)
        heads = qkv.view(T, 3, H, 64)
        q, k = heads[:, 0], heads[:, 1]
        ops.qk_norm_rope(q, k, q, k, K.NORM_RMS, *dh, None, None, dc, ds, None, True, 1e-6, q_scale)
        ops.attention(qkv, o, L)
        ops.quant_mx4(o, codes2, scale2)
        ops.gemm_mx4(codes2, scale2, *weights[1], dbias[1], out, K.EPI_RESIDUAL, 0, x)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        forward()
    torch.cuda.current_stream().wait_stream(side)
    assert_same_mx4((codes, scale), OX.quant_mx4(back, True, OX.LAYER, 0, g, b))
    a = codes.cpu().numpy(), scale.cpu().numpy()
    y, size = OX.gemm_mx4(a, [t.cpu().numpy() for t in weights[0]], bias[0])
    e = sum_error(C, size)
    assert (np.abs(plain.double().cpu().numpy() - y) <= e + HALF["fp16"] * (np.abs(y) + e) + TINY["fp16"]).all()
    p = plain.float().cpu().numpy().reshape(T, 3, H, 64)
    rot = qkv.double().cpu().numpy().reshape(T, 3, H, 64)
    for i, s in ((0, q_scale), (1, 1.0)):
        check_qk(rot[:, i], p[:, i], OQ.RMS, hg[i], None, cos, sin, np.arange(T) % L, True, s, "fp16")
    assert np.array_equal(rot[:, 2], p[:, 2])
    att = OA.attention(qkv.cpu().numpy(), L)
    assert np.abs(o.double().cpu().numpy() - att).max() < 4e-3  # the attention kernel's own bar
    assert_same_mx4((codes2, scale2), OX.quant_mx4(o.float().cpu().numpy()))
    y, size = OX.gemm_mx4((codes2.cpu().numpy(), scale2.cpu().numpy()), [t.cpu().numpy() for t in weights[1]], bias[1])
    want = y + back
    e = sum_error(C, size) + 2.0**-23 * np.abs(want)
    assert (np.abs(out.double().cpu().numpy() - want) <= e + HALF["fp16"] * (np.abs(want) + e) + TINY["fp16"]).all()

    eager = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        forward()
    for i in range(4):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), f"replay {i}"
        forward()  # eager work between the replays
        assert torch.equal(out, eager)


def test_ops_on_two_streams_at_once(dev, rng):
    """The entries keep no state: two products and norms in flight on two streams give what each gives alone."""
    K = kern()
    jobs = []
    for M, N, Kd in ((700, 900, 1024), (65, 2000, 2816)):
        a, w = ([gpu(t, dev) for t in random_mx4(rng, n, Kd, 118, 130)] for n in (M, N))
        jobs.append((a, w, torch.empty(M, N, device=dev)))
    want = []
    for a, w, out in jobs:
        K.gemm_mx4(*a, *w, None, out, K.EPI_BIAS_F16)
        want.append(out.clone())
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(5):
        for (a, w, out), s in zip(jobs, streams):
            with torch.cuda.stream(s):
                out.zero_()
                K.gemm_mx4(*a, *w, None, out, K.EPI_BIAS_F16)
    torch.cuda.synchronize()
    for (_, _, out), ref in zip(jobs, want):
        assert torch.equal(out, ref)


def test_mx4_ops_refuse_tensors_with_a_tangent(dev):
    """Through the dispatcher as well."""
    from torch.autograd import forward_ad

    K = kern()
    x = torch.zeros(2, 128, dtype=torch.half, device=dev)
    codes, scale, _ = empty_mx4(2, 128, dev)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for op in (K.quant_mx4, K.kernels().quant_mx4):
            with pytest.raises(RuntimeError, match="forward mode"):
                op(dual, codes, scale)
            op(x, codes, scale)


@pytest.mark.parametrize("T", [1, 6])
@pytest.mark.parametrize("layout", ["packed", "by head", "heads first", "heads first, by token", "into the values",
                                    "one row of keys"])
def test_qk_norm_rope_rows_between_the_other_operands(dev, rng, layout, T):
    """Layouts in which the operands lie between each other's rows and share nothing: as with operands of their own."""
    K = kern()
    H, D = 4, 64
    cos, sin = (gpu(t, dev) for t in tables(rng, 3, D))
    gq, gk = (gpu((1 + 0.1 * rng.standard_normal(D)).astype(np.float32), dev) for _ in range(2))
    if layout == "one row of keys":
        b, _ = typed(rng.standard_normal((T, H + 1, D)), "fp16", dev)
        q, k = b[:, :H], b[:, H:]
        qo, ko = q, k
    elif layout in ("packed", "into the values"):
        b, _ = typed(rng.standard_normal((T, 4, H, D)), "fp16", dev)
        q, k = b[:, 0], b[:, 1]
        qo, ko = (q, k) if layout == "packed" else (b[:, 2], b[:, 3])
    elif layout == "by head":
        b, _ = typed(rng.standard_normal((T, H, 4, D)), "fp16", dev)
        q, k, qo, ko = (b[:, :, i] for i in range(4))
    elif layout == "heads first":
        b, _ = typed(rng.standard_normal((4, H, T, D)), "fp16", dev)
        q, k, qo, ko = (b[i].transpose(0, 1) for i in range(4))
    else:
        b, _ = typed(rng.standard_normal((H, T, 4, D)), "fp16", dev)
        q, k, qo, ko = (b[:, :, i].transpose(0, 1) for i in range(4))
    want = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty_like(k, memory_format=torch.contiguous_format)
    args = (OQ.RMS, gq, gk, None, None, cos, sin)
    K.qk_norm_rope(q.clone(), k.clone(), *want, *args)
    K.qk_norm_rope(q, k, qo, ko, *args)
    assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])


def test_quant_mx4_outputs_between_the_rows_of_x(dev, rng):
    """Outputs in the memory that the rows of x leave free are taken."""
    K = kern()
    T, C = 5, 128
    x, back = typed(rng.standard_normal((T, C)), "fp16", dev)
    rows = torch.full((T, 512), 7.0, dtype=torch.half, device=dev)
    rows[:, :C] = x
    bytes_ = rows.view(torch.uint8)
    codes = bytes_[1, 2 * C : 2 * C + T * C // 2].view(T, C // 2)
    scale = bytes_[3, 2 * C : 2 * C + 4 * T].view(torch.int32).view(1, T)
    K.quant_mx4(rows[:, :C], codes, scale)
    assert_same_mx4((codes, scale), OX.quant_mx4(back))
    assert torch.equal(rows[:, :C], x)


@pytest.mark.parametrize("norm", [OQ.RMS, OQ.LAYER])
@pytest.mark.parametrize("eps", [2.0**-149, 2.0**-130, 2.0**-126])
def test_qk_norm_rope_with_an_eps_that_is_subnormal(dev, norm, eps):
    """Heads of zeros become beta, heads of +-2^-66 (their mean square, 2^-132, is exact in fp32 and so is its sum with each
    eps: 2^-132 + 2^-149 has 18 bits) and of +-1 are normed: a root of about an ulp, two products and the output's half
    step."""
    K = kern()
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=dev)
    x[1, :, ::2], x[1, :, 1::2] = 2.0**-66, -(2.0**-66)
    x[2, :, ::2], x[2, :, 1::2] = 1.0, -1.0
    one, beta = torch.ones(64, device=dev), torch.full((64,), 0.25, device=dev) if norm == OQ.LAYER else None
    cos, sin = torch.ones(3, 32, device=dev), torch.zeros(3, 32, device=dev)
    o, o2 = torch.empty_like(x), torch.empty_like(x)
    K.qk_norm_rope(x, x, o, o2, norm, one, one, beta, beta, cos, sin, None, True, eps)
    v = x.double()
    want = v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps) + (0.25 if norm == OQ.LAYER else 0.0)
    assert torch.equal(o, o2) and torch.equal(o[0].double(), want[0])
    assert ((o.double() - want).abs() <= (2.0**-8 + 2.0**-20) * want.abs()).all()


# ---- many rows a workgroup, every instantiation, the ends of the exponent range ----


def qk64(x, norm, gamma, beta, cos, sin, pos, pairs, scale):
    """oracle.qk_norm in torch float64 on the GPU: the result and the size of its terms."""
    x = x.double()
    if norm == OQ.LAYER:
        x = x - x.mean(-1, keepdim=True)
    if norm != OQ.NONE:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * gamma.double()
    if norm == OQ.LAYER:
        x = x + beta.double()
    L, half = cos.shape
    ok = (pos >= 0) & (pos < L)
    c, s = (t.double()[torch.where(ok, pos, 0)][:, None] for t in (cos, sin))
    i = torch.arange(half, device=x.device)
    first, second = (2 * i, 2 * i + 1) if pairs else (i, i + half)
    a, b = x[..., first], x[..., second]
    y, size = x.clone(), x.abs()
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    size[..., first], size[..., second] = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
    return torch.where(ok[:, None, None], y * scale, torch.nan), size * abs(scale)


@pytest.mark.parametrize("norm", [OQ.NONE, OQ.RMS, OQ.LAYER])
@pytest.mark.parametrize("pairs", [True, False])
@pytest.mark.parametrize("form", ["rows in order", "int32, in place, 8-byte rows", "int64, in place"])
@pytest.mark.parametrize(("T", "H", "KV", "D", "R", "L"), [
    (20011, 8, 2, 64, 64, 1025), (20011, 8, 2, 64, 48, 1), (30011, 5, 2, 48, 32, 13), (9001, 32, 8, 128, 128, 700),
    (12007, 7, 7, 96, 96, 5000), (9001, 4, 2, 256, 256, 4099)])
def test_qk_norm_rope_many_tokens_a_group(dev, rng, T, H, KV, D, R, L, form, pairs, norm):
    """Three to eleven times as many heads as the resident groups of lanes, so that each group walks over several tokens;
    every token against float64, with check_qk's tolerance. Positions repeat, lie in no order and past both ends."""
    K = kern()
    kind, shift = ("fp16", 0) if form == "rows in order" else ("bf16", 4 if "8-byte" in form else 0)
    g = torch.Generator(device=dev).manual_seed(int(rng.integers(1 << 30)))
    wide = H + 2 * KV
    rows = torch.full((T, wide * D + 8), 7.0, dtype=TYPES[kind], device=dev)
    x = rows[:, shift : shift + wide * D].unflatten(1, (wide, D))
    x.copy_(2 * torch.randn(T, wide, D, device=dev, generator=g) + 0.3)
    q, k = x[:, :H], x[:, H : H + KV]
    gamma = [1 + 0.1 * torch.randn(D, device=dev, generator=g) if norm else None for _ in range(2)]
    beta = [0.1 * torch.randn(D, device=dev, generator=g) if norm == OQ.LAYER else None for _ in range(2)]
    cos, sin = (gpu(t, dev) for t in tables(rng, L, R))
    pos, given = torch.arange(T, device=dev) % L, None
    if form != "rows in order":
        pos = torch.randint(-(L // 8 + 1), L + L // 8 + 1, (T,), device=dev, generator=g)
        given = pos.to(torch.int32 if "int32" in form else torch.int64)
    want = [qk64(t, norm, gamma[i], beta[i], cos, sin, pos, pairs, s) for i, (t, s) in enumerate(((q, 0.37), (k, 1.0)))]
    rest = x[:, H + KV :].clone()
    out = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k)] if given is None else [q, k]
    K.qk_norm_rope(q, k, *out, norm, *gamma, *beta, cos, sin, given, pairs, 1e-6, 0.37)
    for o, (w, size), s in zip(out, want, (0.37, 1.0)):
        o = o.double()
        assert torch.equal(o.isnan(), w.isnan())
        e = 2.0**-17 * (size + (s if norm == OQ.LAYER else 0))
        bad = ((o - w).abs() > e + HALF[kind] * (w.abs() + e) + TINY[kind]).nonzero()
        assert len(bad) == 0, f"{len(bad)} off, first {bad[:4].tolist()}: {o[tuple(bad[0])]} vs {w[tuple(bad[0])]}"
    assert torch.equal(x[:, H + KV :], rest)
    assert (rows[:, :shift] == 7).all() and (rows[:, shift + wide * D :] == 7).all()


def norm_weights(rng, C, c_real, norm):
    g, b = np.zeros(C, np.float32), np.zeros(C, np.float32)
    g[:c_real] = 1 + 0.1 * rng.standard_normal(c_real)
    b[:c_real] = 0.1 * rng.standard_normal(c_real)
    return g, b if norm == OX.LAYER else None


def quant_rows(dev, x, norm, c_real, g, b, rotate=True):
    T, C = x.shape
    codes, scale, check = empty_mx4(T, C, dev)
    kern().quant_mx4(x, codes, scale, rotate, norm, *(None if p is None else gpu(p, dev) for p in (g, b)), c_real)
    assert check(), "wrote outside its outputs"
    return codes, scale


def compare_rows(codes, scale, x, pick, norm, c_real, g, b, rotate=True):
    pick = torch.as_tensor(np.unique(pick), device=x.device)
    assert_same_mx4((codes[pick], scale[:, pick]), OX.quant_mx4(x[pick].float().cpu().numpy(), rotate, norm, c_real, g, b))


@pytest.mark.parametrize("norm", [OX.RMS, OX.LAYER])
@pytest.mark.parametrize("padding", [0, 37, 133])
@pytest.mark.parametrize(("T", "C"), [
    *((4100, c) for c in (128, 384, 640, 896, 1152, 1408, 256, 768, 1280)),  # one and two lane groups a row
    *((6, c) for c in (384, 512, 1024, 1280, 2048, 2560, 2816, 3584, 4096, 4608, 4992, 5632, 6144))])
def test_quant_mx4_norm_every_width(dev, rng, T, C, padding, norm):
    """Each number of lane groups and blocks that the dispatch knows, the row full, padded inside its last block and by more
    than a block, with values in the padding that are not finite."""
    c_real = max(C - padding, 1)
    kind = "bf16" if (C // 128 + padding) % 2 else "fp16"
    x = activations(rng, T, C)
    x[:, c_real:] = rng.choice(np.array([np.inf, -np.inf, np.nan, 5.0], np.float32), (T, C - c_real))
    g, b = norm_weights(rng, C, c_real, norm)
    t = gpu(x, dev).to(TYPES[kind])
    codes, scale = quant_rows(dev, t, norm, c_real, g, b)
    pick = np.concatenate([np.arange(min(T, 40)), np.arange(max(T - 40, 0), T), rng.integers(0, T, 60)])
    compare_rows(codes, scale, t, pick, norm, c_real, g, b)


@pytest.mark.parametrize("norm", [OX.NONE, OX.RMS, OX.LAYER])
@pytest.mark.parametrize(("T", "C", "c_real"), [(100_003, 128, 120), (100_003, 640, 640), (60_001, 768, 700),
                                                (40_003, 512, 512), (40_003, 1024, 1000), (12_007, 2816, 2730),
                                                (9_001, 6144, 6144)])
def test_quant_mx4_more_rows_than_are_resident(dev, rng, T, C, c_real, norm):
    """Each wave walks over several rows: rows of every walk against the oracle, and all of them against calls of 4100 rows,
    in which a wave has one or two."""
    gen = torch.Generator(device=dev).manual_seed(int(rng.integers(1 << 30)))
    c_real = c_real if norm else C
    x = torch.randn(T, C, device=dev, generator=gen)
    x[:, :: 100] *= 20
    x[:, c_real:] = torch.inf
    x = x.half()
    g, b = norm_weights(rng, C, c_real, norm) if norm else (None, None)
    codes, scale = quant_rows(dev, x, norm, c_real, g, b)
    compare_rows(codes, scale, x, np.concatenate([rng.integers(0, T, 120), np.arange(T - 20, T)]), norm, c_real, g, b)
    for at in range(0, T, 4100):
        at = min(at, T - 4100)
        part = quant_rows(dev, x[at : at + 4100], norm, c_real, g, b)
        assert torch.equal(part[0], codes[at : at + 4100]) and torch.equal(part[1], scale[:, at : at + 4100])
    out = torch.empty(T, C, dtype=torch.bfloat16, device=dev)
    kern().dequant_mx4(codes, scale, out)
    pick = torch.as_tensor(rng.integers(0, T, 200), device=dev)
    assert np.array_equal(out[pick].double().cpu().numpy(), OX.values(codes[pick].cpu().numpy(), scale[:, pick].cpu().numpy()))
    for at in range(0, T, 512):
        at = min(at, T - 512)
        part = torch.empty(512, C, dtype=torch.bfloat16, device=dev)
        kern().dequant_mx4(codes[at : at + 512], scale[:, at : at + 512].contiguous(), part)
        assert torch.equal(part, out[at : at + 512])


@pytest.mark.parametrize("rotate", [True, False])
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_quant_mx4_subnormal_values(dev, rng, kind, rotate):
    """Blocks whose largest value is subnormal, in the input's type and in fp32 (bf16: the exponent stops at -127 and the codes
    are what is left), up to ordinary ones."""
    e = np.arange(-24, -8) if kind == "fp16" else np.arange(-134, -118)
    x = (rng.standard_normal((len(e), 256)) * np.exp2(e)[:, None]).astype(np.float32)
    got, want = run_quant(dev, x, kind, rotate, OX.NONE)
    assert_same_mx4(got, want)
    code, ex = OX.unpack(*want)
    assert kind == "fp16" or ((ex[7] == 0).all() and (code[7] & 7).any())  # 2^-127: subnormal, and codes that are not zero


@pytest.mark.parametrize("variant", VARIANTS[1:])
@pytest.mark.parametrize(("ea", "ew"), [
    ([254], [0]), ([0], [254]), ([1], [253]), ([0], [127]), ([127], [0]), ([1], [106]), ([60], [47]), ([254], [114]),
    ([184], [184]), ([254, 0, 254, 0, 10, 240, 100, 100], [0, 254, 0, 254, 244, 14, 154, 154])])
def test_gemm_mx4_ends_of_the_exponents(dev, rng, ea, ew, variant):
    """The two exponents of a product add up to one power of two over the row, ea + ew - 254 = p: every partial sum is a
    multiple of 2^(p - 2) below 36 x 256 x 2^p < 2^(p + 14), so 16 bits hold it, in the range of fp32 (subnormal numbers
    included) for p - 2 >= -149 and p + 14 <= 128: equal to the exact sum."""
    M, N, K = 70, 90, 256
    assert all(-147 <= a + b - 254 <= 114 and a + b == ea[0] + ew[0] for a, b in zip(ea, ew))
    codes = [rng.integers(0, 16, (n, K)).astype(np.uint8) for n in (M, N)]
    a, w = (OX.pack(c, np.tile(np.array(e * 8, np.uint8)[:8], (len(c), 1))) for c, e in zip(codes, (ea, ew)))
    got = run_gemm(dev, a, w, None, "fp32", OG.EPI_BIAS_F16, variant)
    want, _ = OX.gemm_mx4(a, w)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("variant", VARIANTS[1:])
def test_gemm_mx4_sums_past_both_ends(dev, rng, variant):
    """Below half the smallest number: zero, with the bias left to the summation's rounding. One product past the largest:
    infinite, with its sign, in its own element only (the others are the bias: adding zeros is exact)."""
    M, N, K = 40, 36, 384
    codes = [rng.integers(0, 16, (n, K)).astype(np.uint8) for n in (M, N)]
    low = [OX.pack(c, np.full((len(c), K // 32), 40, np.uint8)) for c in codes]  # 36 x 384 x 2^-174
    bias = rng.standard_normal(N).astype(np.float32)
    got = run_gemm(dev, *low, bias, "fp32", OG.EPI_BIAS_F16, variant)
    assert (np.abs(got - bias) <= sum_error(K, np.abs(bias) + 36 * K * 2.0**-174)).all()
    assert not run_gemm(dev, *low, None, "fp32", OG.EPI_BIAS_F16, variant).any()
    one = [np.zeros((n, K), np.uint8) for n in (M, N)]
    one[0][7, 200], one[1][5, 200], one[1][6, 200] = 7, 7, 15  # 6 x 6 and 6 x -6
    high = [OX.pack(c, np.full((len(c), K // 32), 190, np.uint8)) for c in one]  # 36 x 2^126
    got = run_gemm(dev, *high, bias, "fp32", OG.EPI_BIAS_F16, variant)
    want = np.broadcast_to(bias.astype(np.float64), (M, N)).copy()
    want[7, 5], want[7, 6] = np.inf, -np.inf
    assert np.array_equal(got, want)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize(("M", "N"), [(1025, 1030), (300, 768), (513, 771)])
def test_gemm_mx4_residual_in_place_is_the_same(dev, rng, M, N, kind, variant):
    """The residual as out itself, over several tiles in both directions, whole and ragged: bit for bit as from memory of its
    own."""
    K = kern()
    a, w = ([gpu(t, dev) for t in random_mx4(rng, n, 384, 118, 126)] for n in (M, N))
    bias = gpu(rng.standard_normal(N).astype(np.float32), dev)
    x, _ = typed(rng.standard_normal((M, N)), kind, dev)
    out = torch.empty_like(x)
    K.gemm_mx4(*a, *w, bias, out, K.EPI_RESIDUAL, variant, x)
    K.gemm_mx4(*a, *w, bias, x, K.EPI_RESIDUAL, variant)
    assert torch.equal(out, x)


def test_every_op_on_two_streams_at_once(dev, rng):
    """Quantization with a norm, its values, the product and the head norm in flight on two streams, each round into outputs
    of its own: all of them as alone."""
    K = kern()
    cos, sin = (gpu(t, dev) for t in tables(rng, 65, 64))
    one = torch.ones(64, device=dev)
    jobs = []
    for T, C, N, norm in ((1300, 1024, 1280, OX.LAYER), (4100, 640, 512, OX.RMS)):
        x, _ = typed(activations(rng, T, C), "fp16", dev)
        g, b = norm_weights(rng, C, C, norm)
        w = [gpu(t, dev) for t in random_mx4(rng, N, C, 118, 124)]
        jobs.append((x, norm, gpu(g, dev), None if b is None else gpu(b, dev), w))

    def outputs(job):
        (T, C), N = job[0].shape, job[4][0].shape[0]
        return (torch.zeros(T, C // 2, dtype=torch.uint8, device=dev), torch.zeros(C // 128, T, dtype=torch.int32, device=dev),
                torch.zeros(T, C, dtype=torch.half, device=dev), torch.zeros(T, N, dtype=torch.half, device=dev),
                torch.zeros(T, N // 128, 64, dtype=torch.half, device=dev),
                torch.zeros(T, N // 128, 64, dtype=torch.half, device=dev))

    def launch(job, to):
        x, norm, g, b, w = job
        K.quant_mx4(x, to[0], to[1], True, norm, g, b)
        K.dequant_mx4(to[0], to[1], to[2])
        K.gemm_mx4(to[0], to[1], *w, None, to[3], K.EPI_BIAS_F16)
        heads = to[3].view(len(x), 2, -1, 64)
        K.qk_norm_rope(heads[:, 0], heads[:, 1], to[4], to[5], K.NORM_RMS, one, one, None, None, cos, sin)

    want = []
    for job in jobs:
        want.append(outputs(job))
        launch(job, want[-1])
    rounds = [[outputs(job) for job in jobs] for _ in range(6)]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for to in rounds:
        for job, t, s in zip(jobs, to, streams):
            with torch.cuda.stream(s):
                launch(job, t)
    torch.cuda.synchronize()
    for i, to in enumerate(rounds):
        for t, ref in zip(to, want):
            for n, (a, b) in enumerate(zip(t, ref)):
                assert torch.equal(a, b), f"round {i}, output {n}"
