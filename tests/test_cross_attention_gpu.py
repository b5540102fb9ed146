"""Attention to rows of another length and behind a shared prefix on the GPU, against the float64 oracle.

Bar (`bound`): with u half a step of the type, p is rounded once (u of the weighted mean of |v|, called size) and the output
once (u of |o|); x = c q.k is an fp32 sum of D exact products ((D + 4) 2^-23 of sum |q k| c, at most), so p is off by ln 2 times
that and 2 ulp of the exp2, in numerator and denominator; sums over n keys take a rounding per 8 keys in the products (16 at
a time) and 2^-20 for the joints; fp16 weights below 2^-14 of the largest are off by half a subnormal step, 2^-25, each.
"""

from __future__ import annotations

import math

import numpy as np
import pytest

from oracle import cross_attention as OC

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
HALF = {"fp16": 2.0**-11, "bf16": 2.0**-8}


def kern():
    from foidfinder_amd import kernels as K

    return K


def make(rng, kind, dev, *shape, std=1.0):
    t = torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).to(dev).to(TYPES[kind])
    return t, t.float().cpu().numpy()


def guarded(kind, dev, *shape):
    """An output between guard elements: (out, check)."""
    n = math.prod(shape)
    buf = torch.full((n + 128,), 7.0, dtype=TYPES[kind], device=dev)
    return buf[64 : 64 + n].view(shape), lambda: bool((buf[:64] == 7).all() and (buf[64 + n :] == 7).all())


def bound(kind, scale, o, size, load, vmax, n):
    """Per output element, of n keys at most."""
    D = o.shape[-1]
    u = HALF[kind]
    err_x = (D + 4) * 2.0**-23 * scale * math.log2(math.e) * load
    sub = n * 2.0**-25 * vmax if kind == "fp16" else 0.0
    tiny = 2.0**-25 if kind == "fp16" else 2.0**-133
    return u * (np.abs(o) + size) * (1 + 2.0**-6) + 2 * size * (math.log(2) * err_x + 2.0**-22) \
        + size * (n / 8 * 2.0**-24 + 2.0**-20) + sub + tiny


def assert_near(got, want, tol):
    err = np.abs(got - want)
    worst = np.unravel_index(np.argmax(np.where(np.isnan(err), np.inf, err / tol)), err.shape)
    assert np.isfinite(got).all() and (err <= tol).all(), \
        f"{int((~(err <= tol)).sum())} of {err.size} off, worst at {worst}: {got[worst]} vs {want[worst]}, tol {tol[worst]}"


def run_cross(dev, kind, B, L, S, H, KV, D, *, layout="token", lens=None, mask=None, std=1.0, scale=None, seed=0, junk=None):
    K = kern()
    rng = np.random.default_rng(seed)
    scale = D**-0.5 if scale is None else scale
    q, qn = make(rng, kind, dev, B, L, H, D, std=std)
    if layout == "packed":
        kv, kvn = make(rng, kind, dev, B, S, 2, KV, D, std=std)
        k, v, kn, vn = kv[:, :, 0], kv[:, :, 1], kvn[:, :, 0], kvn[:, :, 1]
    elif layout == "head":
        (k, kn), (v, vn) = (tuple(x.swapaxes(1, 2) for x in make(rng, kind, dev, B, KV, S, D, std=std)) for _ in range(2))
    else:
        (k, kn), (v, vn) = make(rng, kind, dev, B, S, KV, D, std=std), make(rng, kind, dev, B, S, KV, D, std=std)
    ln = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    mk = None if mask is None else torch.from_numpy(mask).to(dev)
    if junk is not None:  # what is not seen holds values that must not get into a sum
        hidden = torch.zeros(B, S, dtype=torch.bool, device=dev)
        if ln is not None:
            hidden |= torch.arange(S, device=dev) >= ln[:, None]
        if mk is not None:
            hidden |= ~mk
        k[hidden], v[hidden] = junk, junk
    out, check = guarded(kind, dev, B, L, H, D)
    need = K.cross_attention_work(q, k)
    work = torch.full((need + 64,), math.nan, dtype=torch.float32, device=dev)
    K.cross_attention(q, k, v, out, scale, ln, mk, work[:need] if need else None)
    torch.cuda.synchronize()
    assert check() and bool(work[need:].isnan().all()), "wrote outside its outputs"
    o, size, load = OC.cross_attention(qn, kn, vn, scale, lens, mask)
    assert_near(out.float().cpu().numpy(), o, bound(kind, scale, o, size, load, np.abs(vn).max(initial=0.0), S))
    return need


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("shape", [
    (1, 1, 1, 1, 1, 8), (2, 1, 63, 2, 1, 64), (1, 3, 64, 4, 2, 32), (2, 5, 65, 3, 3, 48), (1, 33, 129, 2, 2, 72),
    (1, 64, 100, 2, 1, 80), (1, 65, 31, 1, 1, 96), (1, 129, 200, 1, 1, 128), (2, 40, 300, 4, 1, 104), (1, 100, 33, 2, 1, 88),
    (3, 1, 1025, 8, 2, 128), (1, 7, 2000, 16, 1, 16), (1, 300, 130, 1, 1, 24), (1, 32, 64, 2, 2, 64), (1, 128, 128, 1, 1, 56),
])
def test_cross_attention_shapes(dev, kind, shape):
    run_cross(dev, kind, *shape)


@pytest.mark.parametrize("layout", ["packed", "head"])
@pytest.mark.parametrize("dim", [40, 64, 96, 128])
def test_cross_attention_layouts(dev, layout, dim):
    run_cross(dev, "bf16", 2, 9, 150, 6, 3, dim, layout=layout)
    run_cross(dev, "fp16", 2, 1, 700, 6, 3, dim, layout=layout)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("junk", [None, math.nan, math.inf])
@pytest.mark.parametrize("L", [1, 20, 70, 140])
def test_cross_attention_lengths(dev, kind, junk, L):
    # none, one, the ends of tiles and halves, all, and values outside 0 .. S
    run_cross(dev, kind, 9, L, 200, 2, 1, 64, lens=[0, 1, 31, 32, 64, 65, 200, 999, -5], junk=junk)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("junk", [None, math.nan])
@pytest.mark.parametrize("L,S,D", [(1, 500, 128), (20, 330, 64), (70, 200, 96), (140, 200, 48)])
def test_cross_attention_masks(dev, kind, junk, L, S, D):
    rng = np.random.default_rng(3)
    mask = rng.random((6, S)) < 0.5
    mask[0] = False                 # nothing left
    mask[1, :130] = False           # whole tiles left out at the front
    mask[2, 70:] = False            # and behind
    mask[3] = np.arange(S) == S - 1  # the last key alone
    mask[4] = True
    run_cross(dev, kind, 6, L, S, 4, 2, D, mask=mask, junk=junk)
    run_cross(dev, kind, 6, L, S, 4, 2, D, mask=mask, lens=[5, S, 64, S - 1, 100, 0], junk=junk)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("L", [1, 40, 100])
def test_cross_attention_steep_scores(dev, kind, L):
    """Scores of some hundreds: a few keys take all the weight, and the reference rises again and again."""
    run_cross(dev, kind, 2, L, 900, 2, 1, 64, std=4.0, scale=1.0)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_cross_attention_rising_and_falling_scores(dev, kind):
    """Keys in the order of their scores, both ways: each tile's are above, or below, all before it."""
    K = kern()
    S, D = 1000, 64
    for sign in (1.0, -1.0):
        q = torch.full((1, 2, 1, D), 1.0, dtype=TYPES[kind], device=dev)
        ramp = sign * torch.linspace(-40, 40, S, device=dev)
        k = (ramp[:, None] / D).expand(S, D).to(TYPES[kind]).view(1, S, 1, D).contiguous()
        v, vn = make(np.random.default_rng(1), kind, dev, 1, S, 1, D)
        out = torch.empty_like(q)
        work = torch.empty(K.cross_attention_work(q, k), device=dev)
        K.cross_attention(q, k, v, out, 1.0, None, None, work)
        qn, kn = q.float().cpu().numpy(), k.float().cpu().numpy()
        o, size, load = OC.cross_attention(qn, kn, vn, 1.0)
        assert_near(out.float().cpu().numpy(), o, bound(kind, 1.0, o, size, load, np.abs(vn).max(), S))


@pytest.mark.parametrize("L", [1, 40, 100])
def test_cross_attention_scores_of_any_size(dev, L):
    """Scores of 2 10^11, whose spacing in fp32 is far above 1, and their negatives: the largest keys, all alike, share the weight.
    Equal scores have equal weights, so their mean is off by the roundings of one weight and of the output."""
    K = kern()
    for sign in (1.0, -1.0):
        q = torch.full((1, L, 1, 64), 60000.0, dtype=torch.float16, device=dev)
        k = torch.full((1, 700, 1, 64), sign * 60000.0, dtype=torch.float16, device=dev)
        k[:, 1::3] = sign * (30000.0 if sign > 0 else 64000.0)
        v, vn = make(np.random.default_rng(2), "fp16", dev, 1, 700, 1, 64)
        out = torch.empty_like(q)
        K.cross_attention(q, k, v, out, 1.0, None, None, torch.empty(max(1, K.cross_attention_work(q, k)), device=dev))
        top = vn[0, np.arange(700) % 3 != 1, 0].astype(np.float64)
        o, size = top.mean(0), np.abs(top).mean(0)
        err = np.abs(out[0, :, 0].float().cpu().numpy() - o)
        assert (err <= HALF["fp16"] * (np.abs(o) + 2 * size)).all(), err.max()


def test_cross_attention_of_one_key_that_is_not_finite(dev):
    """The rows behind the last key repeat none of it: an infinite value comes out as such."""
    q = torch.randn(1, 2, 2, 64, device=dev).half()
    k, v = torch.randn(1, 1, 2, 64, device=dev).half(), torch.full((1, 1, 2, 64), math.inf, device=dev).half()
    out = torch.empty_like(q)
    kern().cross_attention(q, k, v, out, 0.125)
    assert bool((out == math.inf).all())
    q = torch.randn(1, 70, 2, 64, device=dev).half()
    out = torch.empty_like(q)
    kern().cross_attention(q, k, v, out, 0.125)
    assert bool((out == math.inf).all())
    five = torch.randn(1, 1, 2, 64, device=dev).half().expand(1, 5, 2, 64)  # one row five times
    kern().cross_attention(q, five, five, out, 0.125)
    # equal weights: off by the roundings of a weight, of their sum and of the output
    assert bool(((out - five[:, :1]).abs() <= 3 * HALF["fp16"] * five[:, :1].abs() + 2.0**-24).all())


def test_cross_attention_cut_keys(dev):
    """Few rows and many keys: the keys are cut, with lengths that leave cuts empty."""
    need = run_cross(dev, "fp16", 1, 1, 9000, 2, 1, 64)
    assert need > 0
    assert run_cross(dev, "bf16", 4, 2, 3000, 2, 1, 128, lens=[0, 1, 200, 3000]) > 0
    assert run_cross(dev, "bf16", 2, 3, 3000, 1, 1, 96, mask=np.arange(6000).reshape(2, 3000) % 1000 < 3) > 0


def test_cross_attention_of_no_keys_and_no_rows(dev):
    K = kern()
    q = torch.randn(2, 3, 4, 64, device=dev).half()
    k = torch.empty(2, 0, 2, 64, device=dev).half()
    out = torch.full_like(q, 7.0)
    K.cross_attention(q, k, k, out, 0.125)
    assert bool((out == 0).all())
    for e in (q[:0], q[:, :0]):
        K.cross_attention(e, k[: e.size(0)], k[: e.size(0)], out[: e.size(0), : e.size(1)], 0.125)


def test_cross_attention_shared_rows_and_strided_outputs(dev):
    """Queries and keys expanded over the batch, and an output between other rows."""
    K = kern()
    rng = np.random.default_rng(5)
    q, qn = make(rng, "fp16", dev, 1, 3, 4, 64)
    k, kn = make(rng, "fp16", dev, 1, 90, 4, 64)
    v, vn = make(rng, "fp16", dev, 3, 90, 4, 64)
    wide = torch.full((3, 3, 2, 4, 64), 7.0, dtype=torch.float16, device=dev)
    out = wide[:, :, 1]
    work = torch.empty(K.cross_attention_work(q.expand(3, -1, -1, -1), k.expand(3, -1, -1, -1)), device=dev)
    K.cross_attention(q.expand(3, -1, -1, -1), k.expand(3, -1, -1, -1), v, out, 0.125, None, None, work)
    o, size, load = OC.cross_attention(np.repeat(qn, 3, 0), np.repeat(kn, 3, 0), vn, 0.125)
    assert_near(out.float().cpu().numpy(), o, bound("fp16", 0.125, o, size, load, np.abs(vn).max(), 90))
    assert bool((wide[:, :, 0] == 7).all())


def test_cross_attention_offsets_past_32_bits(dev):
    """Tokens 2^23 elements apart: 300 of them span 5 GB."""
    K = kern()
    rng = np.random.default_rng(6)
    S, D, step = 300, 64, 1 << 23
    buf = torch.empty(S * step, dtype=torch.float16, device=dev)
    kv = buf.view(S, step)[:, : 2 * D].view(S, 2, D)
    new, kvn = make(rng, "fp16", dev, S, 2, D)
    kv.copy_(new)
    k, v = kv[None, :, :1], kv[None, :, 1:]
    q, qn = make(rng, "fp16", dev, 1, 40, 1, D)
    out = torch.empty_like(q)
    work = torch.empty(K.cross_attention_work(q, k), device=dev)
    K.cross_attention(q, k, v, out, 0.125, None, None, work)
    o, size, load = OC.cross_attention(qn, kvn[None, :, :1], kvn[None, :, 1:], 0.125)
    assert_near(out.float().cpu().numpy(), o, bound("fp16", 0.125, o, size, load, np.abs(kvn).max(), S))


def run_prefix(dev, kind, B, L, P, S, H, KV, D, *, lens=None, layout="head", std=1.0, seed=0, junk=None):
    K = kern()
    rng = np.random.default_rng(seed)
    q, qn = make(rng, kind, dev, B, L, H, D, std=std)
    (pk, pkn), (pv, pvn) = (make(rng, kind, dev, P, KV, D, std=std) for _ in range(2))
    if layout == "head":
        (k, kn), (v, vn) = (tuple(x.swapaxes(1, 2) for x in make(rng, kind, dev, B, KV, S, D, std=std)) for _ in range(2))
    else:
        (k, kn), (v, vn) = (make(rng, kind, dev, B, S, KV, D, std=std) for _ in range(2))
    ln = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    if junk is not None:
        hidden = torch.arange(S, device=dev) >= ln[:, None]
        k[hidden], v[hidden] = junk, junk
    out, check = guarded(kind, dev, B, L, H, D)
    need = K.prefix_attention_work(q, pk, k)
    work = torch.full((need + 64,), math.nan, dtype=torch.float32, device=dev)
    K.prefix_attention(q, pk, pv, k, v, out, D**-0.5, ln, work[:need])
    torch.cuda.synchronize()
    assert check() and bool(work[need:].isnan().all()), "wrote outside its outputs"
    o, size, load = OC.prefix_attention(qn, pkn, pvn, kn, vn, D**-0.5, lens)
    top = max(np.abs(vn).max(initial=0.0), np.abs(pvn).max(initial=0.0))
    assert_near(out.float().cpu().numpy(), o, bound(kind, D**-0.5, o, size, load, top, P + S))


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("shape", [
    (1, 1, 1, 1, 1, 1, 8), (2, 1, 100, 16, 4, 1, 64), (3, 5, 65, 5, 2, 2, 48), (5, 1, 1025, 70, 4, 2, 128),
    (2, 40, 64, 130, 2, 1, 96), (1, 130, 31, 200, 1, 1, 64), (3, 33, 200, 33, 2, 1, 72), (40, 1, 70, 3, 8, 2, 128),
    (2, 3, 0, 9, 2, 1, 64), (2, 3, 9, 0, 2, 1, 64), (1, 2, 0, 0, 1, 1, 64), (2, 70, 5, 40, 1, 1, 80),
])
def test_prefix_attention_shapes(dev, kind, shape):
    run_prefix(dev, kind, *shape)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("L", [1, 6, 50])
@pytest.mark.parametrize("P", [0, 80])
def test_prefix_attention_lengths(dev, kind, L, P):
    """Lengths shorter than the new tokens leave the first of them the prefix alone, or nothing."""
    run_prefix(dev, kind, 7, L, P, 150, 4, 2, 64, lens=[0, 1, 5, 64, 65, 150, 400], junk=math.nan)


def test_prefix_attention_token_layout_and_steep_scores(dev):
    run_prefix(dev, "bf16", 3, 4, 300, 90, 4, 2, 64, layout="token")
    run_prefix(dev, "fp16", 3, 1, 700, 300, 4, 4, 64, lens=[1, 150, 300], std=6.0)


def test_prefix_attention_is_attention_to_the_joined_rows(dev):
    """One sequence: the same as attention to prefix and own rows in one, with a query that sees all."""
    K = kern()
    g = torch.Generator(device=dev).manual_seed(0)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g).half()  # noqa: E731
    q, k, v = rnd(1, 1, 8, 64), rnd(1, 500, 2, 64), rnd(1, 500, 2, 64)
    a, b = torch.empty_like(q), torch.empty_like(q)
    work = torch.empty(max(K.cross_attention_work(q, k), K.prefix_attention_work(q, k[0, :200], k[:, 200:])), device=dev)
    K.cross_attention(q, k, v, a, 0.125, None, None, work)
    K.prefix_attention(q, k[0, :200], v[0, :200], k[:, 200:], v[:, 200:], b, 0.125, None, work)
    # either is within its own bar of the exact value: twice u (|o| + size), size <= max |v|
    assert bool(((a - b).abs().float() <= 2 * HALF["fp16"] * (a.float().abs() + v.float().abs().amax())).all())


def test_attention_on_streams_and_in_graphs(dev):
    """A captured call replayed over new inputs, with eager calls and synchronizations between, gives the eager call's bits."""
    K = kern()
    g = torch.Generator(device=dev).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g).bfloat16()  # noqa: E731
    q, k, v = rnd(3, 2, 8, 128), rnd(3, 700, 2, 128), rnd(3, 700, 2, 128)
    pk, pv = rnd(300, 2, 128), rnd(300, 2, 128)
    lens = torch.tensor([700, 3, 256], dtype=torch.int32, device=dev)
    outs = [torch.empty_like(q) for _ in range(4)]
    works = [torch.empty(max(K.cross_attention_work(q, k), K.prefix_attention_work(q, pk, k)), device=dev) for _ in range(2)]

    def both(a, b, work):
        K.cross_attention(q, k, v, a, 0.09, lens, None, work)
        K.prefix_attention(q, pk, pv, k, v, b, 0.09, lens, work)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(outs[0], outs[1], works[0])
    torch.cuda.current_stream().wait_stream(side)
    both(outs[2], outs[3], works[1])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both(outs[0], outs[1], works[0])
    for n in range(4):
        for t in (q, k, v, pk, pv):
            t.copy_(rnd(*t.shape))
        lens.copy_(torch.tensor([n, 700 - n, 64 * n], dtype=torch.int32, device=dev))
        graph.replay()
        both(outs[2], outs[3], works[1])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3]), n
