"""MX4 and the head norm without a GPU: the oracles pinned against definitions, and every refusal of the entry points (they
come before any HIP call)."""

from __future__ import annotations

import ctypes
from fractions import Fraction

import numpy as np
import pytest
import torch

from foidfinder_amd import kernels as K
from oracle import mx4 as OX
from oracle import qk_norm as OQ
from oracle.gemm import fma32

FF_OK, FF_EINVAL = 0, 1
ALL_VALUES = [s * g for g in OX.GRID for s in (1, -1)]


def err(status):
    return status, K.lib().ff_last_error().decode()


def test_encode_picks_the_nearest_value_and_the_even_code_on_ties():
    rng = np.random.default_rng(0)
    v = rng.standard_normal((64, 32)).astype(np.float32) * np.exp2(rng.integers(-20, 20, (64, 1))).astype(np.float32)
    v[0] = np.arange(32) * 0.25  # every midpoint of the grid at exponent 0 (the largest value, 7.75, in [4, 8))
    v[1] = -v[0]
    code, e = OX.encode(v)
    for r in range(64):
        top = float(np.abs(v[r]).max())
        unit = 2.0 ** (int(e[r, 0]) - 127)
        assert 4 * unit <= top < 8 * unit
        for x, c in zip(v[r].tolist(), code[r].tolist()):
            m = abs(x) / unit
            d = [abs(m - g) for g in OX.GRID]
            best = [i for i, t in enumerate(d) if t == min(d)]
            want = best[0] if len(best) == 1 else next(i for i in best if i % 2 == 0)
            if m > 6:
                want = 7
            assert c & 7 == want and (c >> 3 == 1) == (np.signbit(x)), (x, c, want)


def test_encode_of_zeros_subnormals_and_values_that_are_not_finite():
    v = np.zeros((1, 160), np.float32)
    v[0, 32] = 2.0**-130
    v[0, 64] = np.inf
    v[0, 96] = np.nan
    v[0, 128] = np.finfo(np.float32).max
    code, e = OX.encode(v)
    assert e[0].tolist() == [0, 0, 255, 255, 252]
    assert not code[0, :32].any() and code[0, 32] == 0  # 2^-130 / 2^-127 = 1/8 rounds to 0
    vals = OX.values(*OX.pack(np.pad(code, ((0, 0), (0, 96))), np.pad(e, ((0, 0), (0, 3)))))
    assert np.isnan(vals[0, 64:128]).all() and vals[0, 128] == 6 * 2.0**125 and not vals[0, :64].any()


def test_pack_puts_even_columns_low_and_four_exponents_in_a_word():
    code = np.arange(256, dtype=np.uint8).reshape(1, 256) % 16
    codes, scale = OX.pack(code, np.arange(8, dtype=np.uint8).reshape(1, 8) + 100)
    assert codes[0, 0] == 0x10 and codes[0, 1] == 0x32 and scale.shape == (2, 1)
    assert scale[1, 0] == 104 | 105 << 8 | 106 << 16 | 107 << 24
    back = OX.unpack(codes, scale)
    assert np.array_equal(back[0], code) and back[1][0].tolist() == list(range(100, 108))


def test_fused_multiply_add_of_infinities_in_the_oracle():
    inf, nan = np.float32(np.inf), np.float32(np.nan)
    with np.errstate(invalid="ignore"):
        got = fma32(np.array([inf, 2, inf, nan, 3e38, 1], np.float32), np.array([inf, 3, 0, 1, 10, 1], np.float32),
                    np.array([1, -inf, 1, 1, 0, inf], np.float32))
    assert np.array_equal(got, np.array([inf, -inf, nan, nan, inf, inf], np.float32), equal_nan=True)


def test_norm_of_a_row_with_an_infinity():
    """RMS: 1 / sqrt(inf) = 0, so finite columns become zeros and the infinite one undefined; the next row is as without."""
    x = np.ones((2, 256), np.float32)
    x[0, 3] = np.inf
    with np.errstate(invalid="ignore"):
        v = OX.norm_rows(x, OX.RMS, 256, np.ones(256, np.float32), None, 1e-6)
    assert np.isnan(v[0, 3]) and not v[0, :3].any() and not v[0, 4:].any()
    assert np.array_equal(v[1], OX.norm_rows(x[1:], OX.RMS, 256, np.ones(256, np.float32), None, 1e-6)[0])


@pytest.mark.parametrize("norm", [OX.RMS, OX.LAYER])
@pytest.mark.parametrize(("C", "c_real"), [(128, 1), (640, 640), (1024, 1000), (2816, 2730)])
def test_norm_rows_against_float64(norm, C, c_real):
    """A sum of n terms in 64 partial sums is off by at most (n / 64 + 6) 2^-24 of the sum of magnitudes: with the mean's
    and the variance's quotient, root and products (1/2 ulp each, under ten of them) a value is off by (C / 32 + 32) 2^-24
    of the row's largest normed value at most."""
    rng = np.random.default_rng(C + norm)
    x = rng.standard_normal((5, C)).astype(np.float32)
    g = np.where(np.arange(C) < c_real, 1 + 0.1 * rng.standard_normal(C), 0).astype(np.float32)
    b = np.where(np.arange(C) < c_real, 0.1 * rng.standard_normal(C), 0).astype(np.float32) if norm == OX.LAYER else None
    got = OX.norm_rows(x, norm, c_real, g, b, 1e-6)
    want = np.zeros((5, C))
    want[:, :c_real] = OQ.head_norm(x[:, :c_real], norm, g[:c_real], None if b is None else b[:c_real], 1e-6)
    assert not got[:, c_real:].any()
    assert np.abs(got - want).max() <= (C / 32 + 32) * 2.0**-24 * max(1.0, np.abs(want).max())


def test_rotation_equals_the_hadamard_product():
    """Seven stages, one rounding of at most half an ulp each, and the factor's: 8 * 2^-24 of the sum of magnitudes."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((4, 256)).astype(np.float32)
    i = np.arange(128)
    h = np.array([[(-1.0) ** bin(a & b).count("1") for b in i] for a in i]) / np.sqrt(128.0)
    v = OX.fwht_rows(x.reshape(-1, 128), tuple(range(7))) * OX.INV_SQRT_128
    want = x.reshape(-1, 128).astype(np.float64) @ h
    assert np.abs(v - want).max() <= 9 * 2.0**-24 * np.abs(x).reshape(-1, 128).sum(1).max() / np.sqrt(128.0)
    codes, scale = OX.quant_mx4(x)
    back = OX.values(codes, scale)
    # a value is off by half a spacing: 1/2 under 4, 1 up to 6, and saturation (6 for values under 8): 2 units of 2^e
    unit = np.repeat(np.ldexp(1.0, OX.unpack(codes, scale)[1].astype(int) - 127), 32, axis=1)
    assert (np.abs(back - v.reshape(4, 256)) <= 2 * unit).all()


def test_gemm_oracle_against_rationals():
    rng = np.random.default_rng(5)
    a, w = (OX.pack(rng.integers(0, 16, (n, 128)).astype(np.uint8), rng.integers(60, 190, (n, 4)).astype(np.uint8))
            for n in (2, 3))
    bias = rng.standard_normal(3).astype(np.float32)
    y, size = OX.gemm_mx4(a, w, bias)
    (ac, ae), (wc, we) = OX.unpack(*a), OX.unpack(*w)

    def val(c, e):
        return Fraction(float(OX.GRID[c & 7])) * (-1 if c & 8 else 1) * Fraction(2) ** (int(e) - 127)

    for m in range(2):
        for n in range(3):
            s = sum(val(ac[m, k], ae[m, k // 32]) * val(wc[n, k], we[n, k // 32]) for k in range(128))
            assert abs(float(s + Fraction(float(bias[n]))) - y[m, n]) <= 1e-13 * size[m, n]


@pytest.mark.parametrize("pairs", [True, False])
def test_rotation_oracle_is_a_complex_product(pairs):
    rng = np.random.default_rng(7)
    x = rng.standard_normal((3, 2, 24))
    ang = rng.uniform(-4, 4, (5, 8))
    pos = np.array([0, 4, 2])
    ang[0] = 0
    y, _ = OQ.qk_norm_rope(x, OQ.NONE, None, None, 1e-6, np.cos(ang), np.sin(ang), pos, pairs, 3.0)
    for t in range(3):
        for i in range(8):
            a, b = (2 * i, 2 * i + 1) if pairs else (i, i + 8)
            z = (x[t, :, a] + 1j * x[t, :, b]) * np.exp(1j * ang[pos[t], i]) * 3
            assert np.allclose(y[t, :, a], z.real, atol=1e-14) and np.allclose(y[t, :, b], z.imag, atol=1e-14)
    assert np.array_equal(y[..., 16:], x[..., 16:] * 3) and np.allclose(y[0], x[0] * 3)
    n, _ = OQ.qk_norm_rope(x, OQ.RMS, np.ones(24), None, 1e-12, np.cos(ang), np.sin(ang), np.array([0, 5, -1]), pairs)
    assert np.allclose((n[0] ** 2).mean(-1), 1) and np.isnan(n[1:]).all()


# ---- refusals of the C entries ----


def test_quant_mx4_rejects_bad_arguments():
    def call(x=256, dtype=0, T=4, C=1024, xs=1024, rotate=1, norm=0, c_real=1024, g=None, b=None, eps=1e-6, out=256, s=256):
        return err(K.lib().ff_quant_mx4(x, dtype, T, C, xs, rotate, norm, c_real, g, b, eps, out, s, None))

    assert call(T=0, x=None) == (FF_OK, "")
    for kw, what in ((dict(dtype=2), "fp16 or bf16"), (dict(T=-1), "T"), (dict(T=1 << 31), "T"), (dict(C=0, xs=0), "C"),
                     (dict(C=1000), "C"), (dict(C=6272, xs=6272), "C"), (dict(xs=1016), "x_stride"),
                     (dict(xs=1028), "x_stride"), (dict(rotate=2), "rotate"), (dict(norm=3), "norm"),
                     (dict(norm=1), "gamma"), (dict(g=256), "gamma"), (dict(norm=2, g=256), "beta"),
                     (dict(norm=1, g=256, b=256), "beta"), (dict(norm=1, g=256, c_real=0), "c_real"),
                     (dict(norm=1, g=256, c_real=1025), "c_real"), (dict(norm=1, g=256, eps=0.0), "eps"),
                     (dict(norm=1, g=256, eps=float("nan")), "eps"), (dict(x=None), "null"), (dict(out=None), "null"),
                     (dict(s=None), "null"), (dict(x=264), "misaligned"), (dict(out=258), "misaligned"),
                     (dict(s=257), "misaligned"), (dict(norm=1, g=260), "misaligned")):
        status, msg = call(**kw)
        assert status == FF_EINVAL and what in msg, (kw, msg)


def test_dequant_mx4_rejects_bad_arguments():
    def call(c=256, s=256, T=4, C=1024, out=256, dtype=0):
        return err(K.lib().ff_dequant_mx4(c, s, T, C, out, dtype, None))

    assert call(T=0, c=None) == (FF_OK, "")
    for kw, what in ((dict(dtype=3), "fp32"), (dict(T=-1), "T"), (dict(C=64), "C"), (dict(c=None), "null"),
                     (dict(s=None), "null"), (dict(out=None), "null"), (dict(out=264), "misaligned"),
                     (dict(c=258), "misaligned"), (dict(s=258), "misaligned")):
        status, msg = call(**kw)
        assert status == FF_EINVAL and what in msg, (kw, msg)


def test_gemm_mx4_rejects_bad_arguments():
    def call(A=256, As=256, W=256, Ws=256, M=8, N=16, Kd=128, bias=256, res=None, out=256, dtype=0, epi=4, variant=0):
        return err(K.lib().ff_gemm_mx4(A, As, W, Ws, M, N, Kd, bias, res, out, dtype, epi, variant, None))

    assert call(M=0, A=None) == (FF_OK, "")
    for kw, what in ((dict(epi=0), "epilogue"), (dict(epi=5), "epilogue"), (dict(dtype=3), "out must"),
                     (dict(dtype=2, epi=2), "out must"), (dict(variant=-1), "variant"), (dict(variant=99), "variant"),
                     (dict(Kd=64), "K must"), (dict(Kd=0), "K must"), (dict(N=0), "N must"), (dict(N=15, epi=3), "even"),
                     (dict(M=-1), "not supported"), (dict(N=(1 << 21) + 1), "not supported"),
                     (dict(Kd=(1 << 22) + 128), "not supported"), (dict(epi=1), "null"), (dict(A=None), "null"),
                     (dict(Ws=None), "null"), (dict(out=None), "null"), (dict(A=264), "misaligned"),
                     (dict(bias=260), "misaligned"), (dict(out=264), "misaligned"), (dict(As=258), "misaligned"),
                     (dict(epi=1, res=264), "misaligned"), (dict(epi=1, res=272), "overlaps"),
                     (dict(M=1 << 29, N=64, variant=1), "too many tiles"),
                     (dict(M=0x7fffff00, N=128, variant=2), "too many tiles"),
                     (dict(M=1 << 29, N=2048, variant=5), "too many tiles"),
                     (dict(epi=1, out=496), "null"), (dict(epi=1, res=256, out=496), "overlaps")):
        status, msg = call(**kw)
        assert status == FF_EINVAL and what in msg, (kw, msg)


def test_qk_norm_rope_rejects_bad_arguments():
    def call(q=256, k=65536, qo=256, ko=65536, st=((1024, 64),) * 4, dtype=0, T=4, H=16, KV=16, D=64, norm=1, g=256, b=None,
             eps=1e-6, cos=256, L=8, R=64, pairs=1, pos=None, pos64=0):
        return err(K.lib().ff_qk_norm_rope(q, *st[0], k, *st[1], qo, *st[2], ko, *st[3], dtype, T, H, KV, D, norm, g, g, b,
                                           b, eps, cos, cos, L, R, pairs, pos, pos64, 1.0, None))

    ok = (1024, 64)
    assert call(T=0, q=None) == (FF_OK, "")
    for kw, what in ((dict(dtype=2), "fp16 or bf16"), (dict(D=60), "heads must"), (dict(D=264), "heads must"),
                     (dict(R=0), "rotated"), (dict(R=60), "rotated"), (dict(R=72), "rotated"), (dict(H=0), "heads"),
                     (dict(KV=65536), "heads"), (dict(T=-1), "T"), (dict(T=1 << 27), "2^31"), (dict(L=0), "rope_len"),
                     (dict(L=1 << 30), "rope_len"), (dict(ko=256), "two"),
                     (dict(q=512, qo=512, k=256, ko=512), "two"), (dict(k=512, qo=512), "two"), (dict(q=65536), "two"),
                     (dict(norm=3), "norm"), (dict(norm=0), "gamma"), (dict(g=None), "gamma"), (dict(b=256), "beta"),
                     (dict(norm=2), "beta"), (dict(eps=0.0), "eps"), (dict(q=None), "null"), (dict(ko=None), "null"),
                     (dict(cos=None), "null"), (dict(q=260), "misaligned"), (dict(cos=264), "misaligned"),
                     (dict(pos=258), "misaligned"), (dict(pos=260, pos64=1), "misaligned"),
                     (dict(st=((1022, 64), ok, ok, ok)), "misaligned"), (dict(st=((-1024, 64), ok, ok, ok)), "negative"),
                     (dict(st=(ok, ok, (960, 64), ok)), "overlap"), (dict(st=(ok, ok, ok, (1024, 56))), "overlap"),
                     (dict(st=(ok, ok, (0, 64), ok)), "overlap"), (dict(st=(ok, ok, (64, 192), ok)), "overlap")):
        status, msg = call(**kw)
        assert status == FF_EINVAL and what in msg, (kw, msg)


def test_python_layer_refuses_wrong_tensors(monkeypatch):
    """The checks of the wrappers, with the device check taken as passed (it comes first and needs a GPU)."""
    monkeypatch.setattr(K, "_on_gpu", lambda *ts: -1)
    monkeypatch.setattr(K, "_run", lambda *a: None)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))

    def mx(T, C):
        return torch.zeros(T, C // 2, dtype=torch.uint8), torch.zeros(C // 128, T, dtype=torch.int32)

    x = torch.zeros(3, 256, dtype=torch.half)
    K.quant_mx4(x, *mx(3, 256))
    K.quant_mx4(torch.zeros(3, 512, dtype=torch.half)[:, :256], *mx(3, 256))
    for bad, out in ((x.float(), mx(3, 256)), (x, mx(3, 128)), (x, mx(4, 256)), (x.t(), mx(256, 128)),
                     (x, (mx(3, 256)[0].int(), mx(3, 256)[1])), (x, (mx(3, 256)[0], mx(3, 256)[1].long()))):
        with pytest.raises(RuntimeError):
            K.quant_mx4(bad, *out)
    with pytest.raises(RuntimeError, match="fp32"):
        K.quant_mx4(x, *mx(3, 256), True, K.NORM_RMS, torch.zeros(128))
    with pytest.raises(RuntimeError, match="backward"):
        K.quant_mx4(x.clone().requires_grad_(), *mx(3, 256))
    with torch.no_grad():
        K.quant_mx4(x.clone().requires_grad_(), *mx(3, 256))
    followed = torch.zeros(3, 256).requires_grad_()
    for call in (lambda: K.dequant_mx4(*mx(3, 256), followed),
                 lambda: K.gemm_mx4(*mx(3, 128), *mx(256, 128), None, followed, K.EPI_BIAS_F16)):
        with pytest.raises(RuntimeError, match="backward"):
            call()
    a, w, o = mx(3, 256), mx(6, 256), torch.zeros(3, 6)
    K.gemm_mx4(*a, *w, None, o, K.EPI_BIAS_F16)
    for call in (lambda: K.gemm_mx4(*a, *mx(6, 128), None, o, K.EPI_BIAS_F16),
                 lambda: K.gemm_mx4(*a, *w, torch.zeros(5), o, K.EPI_BIAS_F16),
                 lambda: K.gemm_mx4(*a, *w, None, o[:, :3], K.EPI_BIAS_F16),
                 lambda: K.gemm_mx4(*a, *w, None, o, K.EPI_SWIGLU),
                 lambda: K.gemm_mx4(*a, *w, None, o, K.EPI_BIAS_F16, 0, o),
                 lambda: K.gemm_mx4(*a, *w, None, o, K.EPI_RESIDUAL, 0, o.half()),
                 lambda: K.dequant_mx4(*a, torch.zeros(3, 128)),
                 lambda: K.dequant_mx4(*a, torch.zeros(3, 256, dtype=torch.double))):
        with pytest.raises(RuntimeError):
            call()
    q, t, g = torch.zeros(5, 4, 64, dtype=torch.half), torch.zeros(7, 32), torch.ones(64)

    def qk(q=q, k=q[:, :2], qo=q.clone(), ko=q[:, :2].clone(), gq=g, gk=g, cos=t, sin=t, pos=None):
        K.qk_norm_rope(q, k, qo, ko, K.NORM_RMS, gq, gk, None, None, cos, sin, pos)

    qk()
    qk(pos=torch.zeros(5, dtype=torch.int32))
    for kw in (dict(k=q[:4]), dict(q=q.float()), dict(qo=q.bfloat16()), dict(ko=q), dict(gq=g[:32]), dict(sin=t[:, :16]),
               dict(cos=t.half(), sin=t.half()), dict(pos=torch.zeros(4, dtype=torch.int64)), dict(pos=torch.zeros(5)),
               dict(qo=q.as_strided((5, 4, 64), (64, 320, 1)))):
        with pytest.raises(RuntimeError):
            qk(**kw)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        monkeypatch.undo()
        K.dequant_mx4(*a, torch.zeros(3, 256))


def test_op_schemas():
    ops = K.kernels()
    assert "Tensor(a!) out, Tensor(b!) scale, bool rotate=True" in str(ops.quant_mx4.default._schema)
    assert "Tensor(a!) out, int epi, int stages=0, Tensor? residual=None" in str(ops.gemm_mx4.default._schema)
    assert "Tensor(a!) q_out, Tensor(b!) k_out, int norm" in str(ops.qk_norm_rope.default._schema)
    assert "Tensor(a!) out" in str(ops.dequant_mx4.default._schema)


def test_tensors_with_a_tangent_are_refused(monkeypatch):
    """A forward-mode dual needs no grad, also under no_grad; the ops would lose its tangent. Inside a level, tensors without
    a tangent are taken."""
    from torch.autograd import forward_ad

    monkeypatch.setattr(K, "_on_gpu", lambda *ts: -1)
    monkeypatch.setattr(K, "_run", lambda *a: None)

    def mx(T, C):
        return torch.zeros(T, C // 2, dtype=torch.uint8), torch.zeros(C // 128, T, dtype=torch.int32)

    def calls(x, y, q):
        t = torch.zeros(3, 32)
        return (lambda: K.quant_mx4(x, *mx(3, 256)), lambda: K.dequant_mx4(*mx(3, 256), x),
                lambda: K.gemm_mx4(*mx(3, 128), *mx(256, 128), None, x, K.EPI_BIAS_F16),
                lambda: K.gemm_mx4(*mx(3, 128), *mx(256, 128), y, torch.zeros(3, 256), K.EPI_BIAS_F16),
                lambda: K.qk_norm_rope(q, q, q.clone(), q.clone(), K.NORM_NONE, None, None, None, None, t, t))

    plain = torch.zeros(3, 256, dtype=torch.half), torch.zeros(256), torch.zeros(3, 4, 64, dtype=torch.half)
    with forward_ad.dual_level():
        duals = [forward_ad.make_dual(t, torch.ones_like(t)) for t in plain]
        for call in calls(*duals):
            with pytest.raises(RuntimeError, match="forward mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward mode"):
                call()
        for call in calls(*plain):
            call()


class Extent(ctypes.Structure):
    """ff::Extent of csrc/common.h."""

    _fields_ = [("at", ctypes.c_uint64), ("n", ctypes.c_int64 * 2), ("pitch", ctypes.c_int64 * 2), ("len", ctypes.c_int64)]

    def bytes(self):
        return {self.at + i * self.pitch[0] + j * self.pitch[1] + b for i in range(self.n[0]) for j in range(self.n[1])
                for b in range(self.len)}


def test_operands_that_share_bytes_by_brute_force():
    """Never apart where a byte is shared; always apart where none is, if the pitches are equal or one operand is a range."""
    fn = K.lib()["_ZN2ff5apartERKNS_6ExtentES2_"]
    fn.argtypes, fn.restype = [ctypes.POINTER(Extent)] * 2, ctypes.c_bool
    rng = np.random.default_rng(11)
    seen = set()
    for _ in range(6000):
        kind = rng.integers(4)
        n = [[int(v) for v in rng.integers(1, 5, 2)] for _ in range(2)]
        pitch = [[int(v) for v in rng.integers(0, 40, 2)] for _ in range(2)]
        if kind == 0:
            pitch[1] = pitch[0]
        elif kind == 1:
            n[1] = [1, 1]
        elif kind == 2:  # one token pitch, heads of their own
            pitch[1][0] = pitch[0][0] = int(rng.integers(20, 90))
        a, b = (Extent(int(rng.integers(100, 180)), (ctypes.c_int64 * 2)(*n[i]), (ctypes.c_int64 * 2)(*pitch[i]),
                       int(rng.integers(1, 9))) for i in range(2))
        got, want = fn(a, b), not (a.bytes() & b.bytes())
        assert got == fn(b, a)
        if kind < 2:
            assert got == want, (kind, n, pitch, a.at, b.at, a.len, b.len)
        else:
            assert want or not got, (kind, n, pitch, a.at, b.at, a.len, b.len)
        seen.add((kind, got, want))
    assert {(k, v, v) for k in range(4) for v in (True, False)} <= seen
    far = 1 << 40  # offsets past 32 bits: the same rows a gigabyte on, then 4 bytes into the last of them
    a = Extent(far, (ctypes.c_int64 * 2)(5, 1), (ctypes.c_int64 * 2)(1 << 31, 0), 128)
    for off, want in ((128, True), ((4 << 31) + 128, True), ((4 << 31) + 124, False), (-128, True), (-124, False),
                      (5 << 31, True), ((4 << 31) - 128, True)):
        assert fn(a, Extent(far + off, (ctypes.c_int64 * 2)(5, 1), (ctypes.c_int64 * 2)(1 << 31, 0), 128)) == want, off


def test_qk_norm_rope_refuses_outputs_that_share_memory():
    """Different workgroups read and write the rows: any byte in common but an output in its input's own place is a race."""
    big = 1 << 30

    def call(q=big, k=2 * big, qo=3 * big, ko=4 * big, st=((1024, 64),) * 4, T=4, H=16, KV=16, D=64, cos=5 * big,
             sin=6 * big, g=7 * big, pos=None, pos64=0):
        return err(K.lib().ff_qk_norm_rope(q, *st[0], k, *st[1], qo, *st[2], ko, *st[3], 0, T, H, KV, D, 1, g, g, None, None,
                                           1e-6, cos, sin, 8, 64, 1, pos, pos64, 1.0, None))

    packed = ((2560, 64),) * 4  # q, k and v of [T, 16 + 16 + 8, 64]
    last = 2 * (4 * 1024 - 1)  # the last value of a [4, 16, 64] operand
    for kw in (dict(qo=big + 128), dict(qo=big - 128), dict(qo=big + 2048),  # a head or a token further in q
               dict(k=big + 2048, qo=big + 128, st=packed),  # q_out ends one head into k
               dict(k=big + 2048, qo=big, ko=big + 2048 + 5120, st=packed),  # k_out one token past k
               dict(ko=3 * big + 128), dict(qo=4 * big + last - 6),  # the outputs share heads, or the last values
               dict(qo=big, k=big + 128, st=((1024, 64), (1024, 64), (1024, 64), (1024, 64)), KV=1),  # k is q's second head
               dict(qo=big, st=((1024, 64), (1024, 64), (2048, 64), (1024, 64))),  # in place with other strides
               dict(ko=2 * big, st=((1024, 64), (0, 64), (1024, 64), (1024, 64))),  # in place of one row for every token
               dict(cos=3 * big + 1024), dict(sin=4 * big - 16), dict(g=3 * big + 2 * 3840), dict(pos=4 * big + last - 6),
               dict(pos=4 * big - 24, pos64=1)):
        status, msg = call(**kw)
        assert status == FF_EINVAL and "overlap" in msg, (kw, msg)


def test_gemm_mx4_refuses_an_out_that_shares_memory():
    big = 1 << 30

    def call(A=big, As=2 * big, W=3 * big, Ws=4 * big, bias=5 * big, res=None, out=6 * big, dtype=0, epi=4):
        return err(K.lib().ff_gemm_mx4(A, As, W, Ws, 100, 64, 256, bias, res, out, dtype, epi, 0, None))

    # out 100 x 64 fp16 12 800 bytes (fp32 25 600, SwiGLU 6 400), A 12 800, its scale 800, W 8 192, its scale 512, bias 256
    for kw in (dict(out=big), dict(out=big + 12784), dict(out=big - 12784), dict(out=2 * big - 12800 + 16),
               dict(As=6 * big + 12796), dict(out=3 * big + 8176), dict(out=3 * big - 12784), dict(out=4 * big + 496),
               dict(bias=6 * big + 12784), dict(bias=6 * big + 25584, dtype=2), dict(out=5 * big + 240, dtype=2),
               dict(out=big - 6384, epi=3), dict(epi=1, res=6 * big, out=6 * big, W=6 * big + 12784),
               dict(epi=1, res=6 * big + 12784), dict(epi=1, res=6 * big - 12784)):
        status, msg = call(**kw)
        assert status == FF_EINVAL and "overlap" in msg, (kw, msg)


def test_quant_and_dequant_mx4_refuse_outputs_that_share_memory():
    big = 1 << 30

    def quant(x=big, xs=256, g=2 * big, b=3 * big, out=4 * big, s=5 * big):
        return err(K.lib().ff_quant_mx4(x, 0, 100, 256, xs, 1, 2, 256, g, b, 1e-6, out, s, None))

    # x 100 rows of 512 bytes, gamma and beta 1024 bytes, codes 12 800, scale 800; the codes do not fit between two rows of x
    for kw in (dict(out=big), dict(out=big - 12796), dict(out=big + 51196), dict(s=big + 51196), dict(s=big - 796),
               dict(s=4 * big + 12796), dict(out=5 * big + 796), dict(g=4 * big + 12784), dict(b=4 * big - 1008),
               dict(g=5 * big + 784), dict(b=5 * big - 1008), dict(x=4 * big - 512, xs=512), dict(s=big + 512, xs=512),
               dict(s=big + 512 - 4, xs=1 << 20), dict(s=big + (99 << 21) - 796, xs=1 << 20)):
        status, msg = quant(**kw)
        assert status == FF_EINVAL and "overlap" in msg, (kw, msg)

    def dequant(c=big, s=2 * big, out=3 * big, dtype=0):
        return err(K.lib().ff_dequant_mx4(c, s, 100, 256, out, dtype, None))

    for kw in (dict(out=big), dict(out=big + 12784), dict(out=big - 51184), dict(out=2 * big + 784),
               dict(s=3 * big + 51196), dict(s=3 * big + 102396, dtype=2), dict(c=3 * big + 102396, dtype=2)):
        status, msg = dequant(**kw)
        assert status == FF_EINVAL and "overlap" in msg, (kw, msg)


def test_no_tokens_in_any_layout(monkeypatch):
    """Empty tensors have one address, none: that is not an output in its input's place with other strides."""
    monkeypatch.setattr(K, "_on_gpu", lambda *ts: -1)
    ran = []
    monkeypatch.setattr(K, "_run", lambda *a: ran.append(a))
    b, t = torch.zeros(0, 4, 3, 64, dtype=torch.half), torch.zeros(3, 32)
    o = torch.zeros(0, 4, 64, dtype=torch.half)
    K.qk_norm_rope(b[:, :, 0], b[:, :, 1], o, o.clone(), K.NORM_NONE, None, None, None, None, t, t)
    K.qk_norm_rope(o, o, b[:, :, 0], b[:, :, 1], K.NORM_NONE, None, None, None, None, t, t)
    assert len(ran) == 2
