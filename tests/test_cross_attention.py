"""Attention to other rows and the residual stream between two norms without a GPU: the oracle pinned against definitions, and
every refusal of the entry points (they come before any HIP call)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from foidfinder_amd import kernels as K
from oracle import cross_attention as OC

FF_OK, FF_EINVAL = 0, 1
INF, NAN = float("inf"), float("nan")


def err(status):
    return status, K.lib().ff_last_error().decode()


def test_oracle_attends_to_what_is_seen():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((2, 3, 4, 8)), rng.standard_normal((2, 9, 2, 8)), rng.standard_normal((2, 9, 2, 8))
    t = [torch.from_numpy(x).transpose(1, 2) for x in (q, k.repeat(2, 2), v.repeat(2, 2))]
    mask = rng.random((2, 9)) < 0.6
    seen = torch.from_numpy(mask & (np.arange(9) < np.array([[9], [5]])))[:, None, None]
    want = torch.nn.functional.scaled_dot_product_attention(*t, attn_mask=seen, scale=0.3).transpose(1, 2).numpy()
    o, size, load = OC.cross_attention(q, k, v, 0.3, [9, 5], mask)
    np.testing.assert_allclose(o, want, rtol=1e-12, atol=1e-13)
    assert (size >= np.abs(o) - 1e-13).all()
    _, _, load = OC.cross_attention(q, k, v, 0.3)
    assert (load[..., 0] >= np.abs(np.einsum("blhd,bshd->blhs", q, k.repeat(2, 2))).max(-1) - 1e-13).all()
    o, _, _ = OC.cross_attention(q, k, v, 0.3, [0, 5], mask & (np.arange(9) > 6))
    assert not o.any()  # no keys left


def test_oracle_prefix_is_causal_behind_the_prefix():
    rng = np.random.default_rng(1)
    q, k, v = rng.standard_normal((1, 3, 2, 8)), rng.standard_normal((1, 6, 1, 8)), rng.standard_normal((1, 6, 1, 8))
    pk, pv = rng.standard_normal((4, 1, 8)), rng.standard_normal((4, 1, 8))
    o, _, _ = OC.prefix_attention(q, pk, pv, k, v, 0.3, [5])
    t = [torch.from_numpy(x) for x in (q[0], np.concatenate((pk, k[0, :5])).repeat(2, 1), np.concatenate((pv, v[0, :5])).repeat(2, 1))]
    seen = torch.arange(9)[None] <= torch.arange(6, 9)[:, None]  # the new tokens are rows 6, 7, 8 of the 9
    want = torch.nn.functional.scaled_dot_product_attention(*(x.transpose(0, 1) for x in t), attn_mask=seen, scale=0.3)
    np.testing.assert_allclose(o[0], want.transpose(0, 1).numpy(), rtol=1e-12, atol=1e-13)


def test_oracle_residual_norm():
    rng = np.random.default_rng(2)
    x, y, g, b = rng.standard_normal((6, 16)), rng.standard_normal((6, 16)), rng.standard_normal(16), rng.standard_normal(16)
    gate = rng.standard_normal((3, 16))
    s, h = OC.residual_norm(x, y, 2, g, b, 1, b, None, gate, 0.5, 1e-3)
    ln = torch.nn.functional.layer_norm(torch.from_numpy(y), (16,), torch.from_numpy(g), torch.from_numpy(b), 1e-3).numpy()
    want = x + 0.5 * gate.repeat(2, 0) * ln
    np.testing.assert_allclose(s, want, rtol=1e-12)
    np.testing.assert_allclose(h, want / np.sqrt((want**2).mean(1, keepdims=True) + 1e-3) * b, rtol=1e-12)


# ---- refusals of the C entries: addresses are never followed ----

Q, KEY, VAL, OUT, WORK, LENS, MASK, PK, PV = (i << 40 for i in range(1, 10))


def cross(q=Q, k=KEY, v=VAL, out=OUT, dtype=0, B=2, L=40, S=100, H=4, KV=2, D=64, scale=0.125, lens=None, mask=None, mb=100,
          work=None, size=0, qs=None, ks=None, vs=None, os=None):
    qs = qs or (L * H * D, H * D, D)
    ks = ks or (S * KV * D, KV * D, D)
    return err(K.lib().ff_cross_attention(q, *qs, k, *ks, v, *(vs or ks), out, *(os or qs), dtype, B, L, S, H, KV, D, scale, lens,
                                          mask, mb, work, size, None))


def prefix(q=Q, pk=PK, pv=PV, k=KEY, v=VAL, out=OUT, dtype=1, B=2, L=1, P=200, S=50, H=4, KV=2, D=64, scale=0.125, lens=None,
           work=WORK, size=1 << 30, ps=None, ks=None):
    qs, ks, ps = (L * H * D, H * D, D), ks or (S * KV * D, KV * D, D), ps or (KV * D, D)
    return err(K.lib().ff_prefix_attention(q, *qs, pk, *ps, pv, *ps, k, *ks, v, *ks, out, *qs, dtype, B, L, P, S, H, KV, D, scale,
                                           lens, work, size, None))


def refused(result, word):
    assert result[0] == FF_EINVAL and word in result[1], result


def test_attention_sizes_and_types_are_checked():
    for call in (cross, prefix):
        for d in (0, -8, 60, 136):
            refused(call(D=d), "columns")
        refused(call(H=0), "heads")
        refused(call(KV=0), "heads")
        refused(call(H=5), "heads")
        refused(call(H=65536, KV=1), "heads")
        refused(call(dtype=2), "fp16 or bf16")
        for s in (0.0, -1.0, INF, NAN):
            refused(call(scale=s), "scale")
        refused(call(B=-1), "negative")
        refused(call(S=-1), "negative")
        refused(call(S=0x7FFFFF01), "keys")
        refused(call(B=1 << 20, L=1 << 10, H=2, KV=2), "2^31")
        refused(call(B=1 << 31), "2^31")
        assert call(B=0) == (FF_OK, "") and call(L=0) == (FF_OK, "")  # nothing to do
    refused(prefix(P=-1), "negative")
    refused(prefix(P=0x7FFFFF01), "keys")
    refused(cross(B=1 << 24, L=1, H=4, KV=4), "too many rows")
    refused(prefix(B=1 << 26, L=1, H=16, KV=1, D=128), "too many rows")


def test_attention_pointers_and_strides_are_checked():
    for call in (cross, prefix):
        for name in ("q", "k", "v", "out"):
            refused(call(**{name: None}), "null")
        for name in ("q", "k", "v"):
            refused(call(**{name: Q + 8}), "misaligned")
        refused(call(out=OUT + 4), "misaligned")
        refused(call(ks=(12800, 132, 64)), "misaligned")
        refused(call(ks=(12800, -128, 64)), "negative")
        refused(call(ks=(12800, 1 << 24, 64)), "2^24")
        refused(call(lens=LENS + 2), "misaligned")
    refused(prefix(pk=None), "null")
    refused(prefix(pv=PV + 8), "misaligned")
    refused(prefix(ps=(1 << 24, 64)), "2^24")
    refused(cross(mask=MASK, mb=-1), "negative")
    refused(cross(os=(10240, 250, 64)), "misaligned")
    refused(cross(os=(10240, 128, 64)), "rows of out overlap")
    refused(cross(os=(0, 256, 64)), "rows of out overlap")
    refused(cross(os=(10240, 256, 0)), "rows of out overlap")


def test_attention_workspace_is_checked():
    assert K.lib().ff_cross_attention_work(64, 1000, 1000, 16, 16, 64) == 0  # enough rows: keys are not cut
    need = K.lib().ff_cross_attention_work(1, 1, 9000, 4, 2, 64)
    assert need > 0
    one = dict(B=1, L=1, S=9000)
    refused(cross(**one), "workspace is too small")
    refused(cross(**one, work=WORK, size=need - 1), "workspace is too small")
    refused(cross(**one, work=None, size=need), "workspace is too small")
    refused(cross(**one, work=WORK + 4, size=need), "misaligned")
    need = K.lib().ff_prefix_attention_work(2, 40, 200, 50, 4, 2, 64)
    assert need > 0
    refused(prefix(L=40, size=need - 1), "workspace is too small")
    refused(prefix(L=40, work=None), "workspace is too small")
    for bad in ((2, 1, -1, 50, 4, 2, 64), (2, 1, 9, 50, 4, 3, 64), (2, 1, 9, 50, 4, 2, 300), (-2, 1, 9, 50, 4, 2, 64)):
        assert K.lib().ff_prefix_attention_work(*bad) == 0


def test_attention_overlaps_are_refused():
    end = 2 * 40 * 4 * 64 * 2  # bytes of q
    for name in ("q", "k", "v"):
        refused(cross(**{name: OUT}), "out overlaps what is read")
        refused(cross(**{name: OUT + end - 16}), "out overlaps what is read")
    refused(cross(lens=OUT + 64), "out overlaps what is read")
    refused(cross(mask=OUT + 64), "out overlaps what is read")
    one = dict(B=1, L=1, S=9000, size=1 << 30)
    refused(cross(**one, work=OUT), "out overlaps the workspace")
    refused(cross(**one, work=KEY), "workspace overlaps what is read")
    refused(cross(**one, work=Q), "workspace overlaps what is read")
    refused(prefix(pk=OUT), "out overlaps what is read")
    refused(prefix(L=40, work=PV), "workspace overlaps what is read")
    # a head-major output laid over a token-major query
    refused(cross(q=OUT, os=(40 * 4 * 64, 64, 40 * 64)), "out overlaps what is read")


def residual(x=Q, y=KEY, xo=OUT, h=VAL, xr=64, yr=64, xor=64, hr=64, dtype=0, T=8, C=64, post=1, pg=PK, pb=None, pre=1, qg=PV,
             qb=None, gate=None, rows=0, gt=0, scale=1.0, eps=1e-6):
    return err(K.lib().ff_residual_norm(x, xr, y, yr, xo, xor, h, hr, dtype, T, C, post, pg, pb, pre, qg, qb, gate, rows, gt,
                                        scale, eps, None))


def test_attention_scale_reaches_the_exponent():
    for call in (cross, prefix):
        refused(call(scale=2.5e38), "scale")  # finite, 2.5e38 log2(e) is not


def test_residual_norm_refusals():
    refused(residual(dtype=2), "fp16 or bf16")
    for c in (0, 60, 16392):
        refused(residual(C=c), "columns")
    refused(residual(T=-1), "T")
    refused(residual(T=1 << 31), "T")
    refused(residual(post=3), "unknown norm")
    refused(residual(post=0), "gamma")
    refused(residual(pg=None), "gamma")
    refused(residual(post=2), "beta")
    refused(residual(qb=WORK), "beta")
    for e in (0.0, -1.0, NAN):
        refused(residual(eps=e), "eps")
    refused(residual(gate=WORK, rows=1, gt=1), "gate must be")
    for n in (0, -1, 3, 16):
        refused(residual(gate=WORK, rows=n), "multiple of the gate's rows")
    for name in ("x", "y", "xo"):
        refused(residual(**{name: None}), "null")
    refused(residual(h=None), "h goes with")
    refused(residual(pre=0, qg=None), "h goes with")
    for name in ("x", "y", "xo", "h", "pg", "qg"):
        refused(residual(**{name: WORK + 8}), "misaligned")
    refused(residual(gate=WORK + 8, rows=1), "misaligned")
    refused(residual(xr=68), "misaligned")
    refused(residual(yr=-64), "negative")
    refused(residual(xor=56), "rows of an output overlap")
    refused(residual(hr=0), "rows of an output overlap")
    refused(residual(xo=VAL), "overlaps")  # both outputs in one place
    refused(residual(xo=Q + 64), "overlaps")  # in place but for some bytes
    refused(residual(xo=Q, xor=72), "overlaps")  # in place with another stride
    for name in ("pg", "qg"):
        refused(residual(**{name: OUT + 32}), "overlaps")
    refused(residual(gate=VAL + 32, rows=1), "overlaps")
    assert residual(T=0) == (FF_OK, "")


def test_python_ops_refuse_what_does_not_fit():
    q = torch.zeros(1, 2, 4, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        K.cross_attention(q, q, q, q, 1.0)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        K.prefix_attention(q, q[0], q[0], q, q, q, 1.0)
    with pytest.raises(RuntimeError, match="one GPU"):
        K.residual_norm(q[0, 0], q[0, 0], q[0, 1], None, 0, None, None, 0, None, None)
    with pytest.raises(RuntimeError, match="no backward"):
        K.cross_attention(q.float().requires_grad_(), q, q, q, 1.0)
    for name, n in (("cross_attention", 5), ("prefix_attention", 7)):
        with pytest.raises((RuntimeError, NotImplementedError)):  # no CPU kernel is registered
            getattr(K.kernels(), name)(*([q] * (n - 1)), 1.0)


def test_cross_attention_of_many_rows_whose_last_round_alone_is_cut():
    """Only the rows of that round are joined: 2^26 rows in all are no limit there."""
    size, few = (8, 524544, 2100, 16, 16, 8), (8, 4352, 2100, 16, 16, 8)
    work = K.lib().ff_cross_attention_work
    assert 8 * 524544 * 16 > 1 << 26
    assert work(*size) == work(*few) > 0  # the same rest of 256 whole row tiles
    refused(cross(B=8, L=524544, S=2100, H=16, KV=16, D=8), "workspace is too small")
    refused(prefix(B=1 << 22, L=1, P=9000, S=9, H=32, KV=1), "too many rows")  # every row is joined
