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


def reference64(q, k, v, scale, seen):
    """The oracle's three values from torch in float64 on the GPU, for shapes that are too large for it: q [B, L, H, D], k, v
    [B, S, KV, D], seen bool [B, L or 1, S] (every query sees a key)."""
    B, L, H, D = q.shape
    G = H // k.size(2)
    out = [torch.empty(B, L, H, n, dtype=torch.float64, device=q.device) for n in (D, D, 1)]
    for b in range(B):
        for h in range(H):
            qq, kk, vv = q[b, :, h].double(), k[b, :, h // G].double(), v[b, :, h // G].double()
            hidden = ~seen[b].expand(L, -1)
            p = torch.softmax((qq @ kk.t().contiguous() * scale).masked_fill(hidden, -math.inf), -1)
            out[0][b, :, h], out[1][b, :, h] = p @ vv, p @ vv.abs()
            load = (qq.abs() @ kk.abs().t().contiguous()).masked_fill(hidden, 0.0)
            out[2][b, :, h] = load.amax(-1, keepdim=True)
    return tuple(t.cpu().numpy() for t in out)


@pytest.mark.parametrize("kind,D,B,H,KV", [("fp16", 64, 9, 16, 16), ("bf16", 128, 2, 32, 1)])
def test_cross_attention_last_round_cut(dev, kind, D, B, H, KV):
    """More row tiles than the chip holds at once, some of them in a last round whose keys are cut, and rows behind the whole tiles."""
    K = kern()
    L, S = 1029, 2100
    g = torch.Generator(device=dev).manual_seed(7)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g).to(TYPES[kind])  # noqa: E731
    q, k, v = rnd(B, L, H, D), rnd(B, S, KV, D), rnd(B, S, KV, D)
    lens = torch.randint(1, S + 1, (B,), device=dev, generator=g).int()
    lens[-1], lens[0] = 3, S  # the tail's sequences among them
    mask = torch.rand(B, S, device=dev, generator=g) < 0.7
    mask[:, 0] = True
    out, check = guarded(kind, dev, B, L, H, D)
    need = K.cross_attention_work(q, k)
    assert 0 < need < B * L * H * (D + 2), "the shape does not cut the last round alone"
    work = torch.full((need + 64,), math.nan, device=dev)
    K.cross_attention(q, k, v, out, D**-0.5, lens, mask, work[:need])
    assert check() and bool(work[need:].isnan().all())
    seen = (mask & (torch.arange(S, device=dev) < lens[:, None]))[:, None]
    o, size, load = reference64(q, k, v, D**-0.5, seen)
    assert_near(out.float().cpu().numpy(), o, bound(kind, D**-0.5, o, size, load, v.float().abs().max().item(), S))


def masked_call(dev, q, k, v, lens, mask, kind):
    """One call with not-a-number in the keys that are not seen, against float64 on the GPU."""
    K = kern()
    B, S, D = k.size(0), k.size(1), k.size(3)
    seen = mask.expand(B, S) & (torch.arange(S, device=dev) < (lens[:, None] if lens is not None else S))
    k[~seen], v[~seen] = math.nan, math.nan
    out, check = guarded(kind, dev, *q.shape)
    need = K.cross_attention_work(q, k)
    work = torch.full((need + 64,), math.nan, device=dev)
    K.cross_attention(q, k, v, out, D**-0.5, lens, mask, work[:need])
    assert check() and bool(work[need:].isnan().all())
    some = seen.any(1)
    k, v = k[some].masked_fill(~seen[some][:, :, None, None], 0), v[some].masked_fill(~seen[some][:, :, None, None], 0)
    o, size, load = reference64(q[some], k, v, D**-0.5, seen[some][:, None])
    got, some = out.float().cpu().numpy(), some.cpu().numpy()
    assert_near(got[some], o, bound(kind, D**-0.5, o, size, load, v.abs().max().item(), S))
    assert (got[~some] == 0).all()


@pytest.mark.parametrize("with_lens", [False, True])
@pytest.mark.parametrize("kind,B,L,S,H,KV,D", [
    ("fp16", 6, 140, 4161, 16, 16, 64),   # rows behind the whole tile that are streamed
    ("bf16", 8, 55, 5000, 24, 8, 96),     # 165 rows: the rest is two units
    ("fp16", 9, 61, 1111, 64, 64, 88),    # two units alone
    ("bf16", 6, 200, 4100, 32, 8, 128), ("fp16", 12, 130, 2500, 16, 16, 40),
    ("bf16", 6, 70, 6000, 1, 1, 128),     # few rows: keys cut, some runs of them without any left
])
def test_cross_attention_of_listed_keys(dev, kind, B, L, S, H, KV, D, with_lens):
    g = torch.Generator(device=dev).manual_seed(11)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g).to(TYPES[kind])  # noqa: E731
    q, kv = rnd(B, L, H, D), rnd(B, S, 2, KV, D)
    at = torch.arange(S, device=dev)
    mask = torch.rand(B, S, device=dev, generator=g) < torch.linspace(0.02, 0.98, B, device=dev)[:, None]
    mask[0] = at == S - 1           # the last alone
    mask[1] = True
    mask[2] = (at >= 70) & (at < S - 70)
    mask[3, 64:] = False            # one whole tile
    lens = None
    if with_lens:
        lens = torch.tensor([S + 9, S - 1, S // 2, 65, *[S - 100] * (B - 4)], dtype=torch.int32, device=dev)
        mask[:, 0] = True
    else:
        mask[5] = False             # nothing left
    masked_call(dev, q, kv[:, :, 0], kv[:, :, 1], lens, mask, kind)


@pytest.mark.parametrize("dim,chunk", [(64, 1024), (96, 512), (128, 2048)])
@pytest.mark.parametrize("tokens", [40, 100])
def test_cross_attention_keys_left_over_chunks_of_the_mask(dev, dim, chunk, tokens):
    """Keys that earlier chunks leave for a later one's first tile: none, fewer than a tile, one, more; in every second chunk."""
    left = [0, 1, 63, 64, 65, 127, 128, chunk - 1, chunk]
    S, B = 5 * chunk + 3, len(left)
    g = torch.Generator(device=dev).manual_seed(14)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g).half()  # noqa: E731
    q, k, v = rnd(B, tokens, 1, dim), rnd(B, S, 1, dim), rnd(B, S, 1, dim)
    mask = torch.zeros(B, S, dtype=torch.bool, device=dev)
    for b, n in enumerate(left):
        for c in (0, 2, 3):
            mask[b, c * chunk + torch.randperm(chunk, device=dev, generator=g)[:n]] = True
        mask[b, S - 1 - b % 3] = True
    masked_call(dev, q, k, v, None, mask, "fp16")


@pytest.mark.parametrize("apart,S", [(131072, 4100), (1 << 22, 600), ((1 << 24) - 8, 200)])
def test_cross_attention_masked_keys_far_apart(dev, apart, S):
    """Up to 32 MiB between a sequence's rows: 64 keys of a list, or fewer, span more than 32-bit offsets reach."""
    L, H, D = 70, 4, 64
    g = torch.Generator(device=dev).manual_seed(12)
    store = torch.empty(S * apart, dtype=torch.float16, device=dev)
    rows = store.view(1, S, apart)[:, :, apart - 2 * H * D :].view(1, S, 2, H, D)
    rows.copy_(torch.randn(1, S, 2, H, D, device=dev, generator=g))
    q = torch.randn(1, L, H, D, device=dev, generator=g).half()
    for kept in (0.05, 0.6):
        mask = torch.rand(1, S, device=dev, generator=g) < kept
        mask[:, -1] = True
        rows.copy_(torch.randn(1, S, 2, H, D, device=dev, generator=g))
        masked_call(dev, q, rows[:, :, 0], rows[:, :, 1], None, mask, "fp16")


def test_cross_attention_masks_captured_and_shared(dev):
    """One mask row for the batch, keys broadcast over it, captured, and replayed over new masks."""
    K = kern()
    B, L, S, H, D = 8, 524, 4161, 16, 64
    g = torch.Generator(device=dev).manual_seed(13)
    q = torch.randn(B, L, H, D, device=dev, generator=g).half()
    one = torch.randn(1, S, 2, H, D, device=dev, generator=g).half()
    k, v = (one[:, :, i].expand(B, -1, -1, -1) for i in range(2))
    row = torch.rand(1, S, device=dev, generator=g) < 0.5
    other = torch.rand(B, S, device=dev, generator=g) < 0.3
    outs = [torch.empty_like(q) for _ in range(4)]
    work = torch.empty(max(1, K.cross_attention_work(q, k)), device=dev)

    def both(a, b, w):
        K.cross_attention(q, k, v, a, 0.125, None, row.expand(B, -1), w)
        K.cross_attention(q, k, v, b, 0.125, None, other, w)

    both(outs[0], outs[1], work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both(outs[0], outs[1], work)
    for n in range(4):
        row.copy_(torch.rand(1, S, device=dev, generator=g) < 0.2 * n)  # nothing left in the first
        other.copy_(torch.rand(B, S, device=dev, generator=g) < 0.9 - 0.2 * n)
        graph.replay()
        both(outs[2], outs[3], torch.full_like(work, math.nan))
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3]), n
        kept = row[0].nonzero()[:, 0]  # the same keys by themselves: the same tiles, for whole tiles of rows
        K.cross_attention(q, k[:, kept], v[:, kept], outs[2], 0.125)
        assert torch.equal(outs[2][:, :512], outs[0][:, :512]) and (n > 0) == bool(outs[0].any()), n


@pytest.mark.parametrize("kind,shape", [
    ("fp16", (70, 4, 40, 20, 8, 4, 64)), ("bf16", (300, 1, 1, 3, 2, 1, 32)), ("fp16", (40, 3, 700, 33, 8, 8, 64)),
    ("bf16", (33, 8, 31, 65, 16, 8, 128)), ("fp16", (90, 2, 330, 100, 3, 3, 96)), ("bf16", (520, 1, 64, 0, 1, 1, 48)),
])
def test_prefix_attention_of_many_sequences_read_by_each(dev, kind, shape):
    """More sequences and key heads than CUs behind a short prefix: one launch, no workspace, the prefix read by each."""
    B, L, _, S = shape[:4]
    rng = np.random.default_rng(21)
    lens = rng.integers(0, S + 1, B)  # some shorter than the new tokens: these see the prefix alone
    lens[:3] = 0, S, S + 7
    K = kern()
    q, pk, k = (torch.empty(s, dtype=torch.float16, device=dev) for s in
                ((B, L, shape[4], shape[6]), (shape[2], shape[5], shape[6]), (B, S, shape[5], shape[6])))
    assert K.prefix_attention_work(q, pk, k) == 0
    run_prefix(dev, kind, *shape, lens=lens.tolist(), junk=math.nan)


@pytest.mark.parametrize("kind,shape", [
    ("fp16", (4, 128, 0, 128, 4, 4, 64)), ("bf16", (2, 45, 0, 700, 4, 2, 128)), ("fp16", (1, 40, 0, 3000, 2, 1, 96)),
    ("bf16", (3, 70, 0, 50, 1, 1, 40)),
])
def test_prefix_attention_without_a_prefix(dev, kind, shape):
    B, S = shape[0], shape[3]
    run_prefix(dev, kind, *shape)
    run_prefix(dev, kind, *shape, lens=[S, 0, S // 2, 1][:B], junk=math.inf)


@pytest.mark.parametrize("kind,B,L,P,S,H,KV,D", [("bf16", 40, 3, 3000, 200, 8, 2, 128), ("fp16", 12, 30, 2000, 900, 16, 16, 64),
                                                 ("fp16", 100, 1, 700, 2500, 4, 4, 96), ("bf16", 3, 200, 64, 5000, 2, 1, 64)])
def test_prefix_attention_of_many_rows_and_cuts(dev, kind, B, L, P, S, H, KV, D):
    K = kern()
    g = torch.Generator(device=dev).manual_seed(8)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g).to(TYPES[kind])  # noqa: E731
    q, pk, pv, k, v = rnd(B, L, H, D), rnd(P, KV, D), rnd(P, KV, D), rnd(B, S, KV, D), rnd(B, S, KV, D)
    lens = torch.randint(L, S + 1, (B,), device=dev, generator=g).int()
    out, check = guarded(kind, dev, B, L, H, D)
    need = K.prefix_attention_work(q, pk, k)
    assert need > 0
    work = torch.full((need + 64,), math.nan, device=dev)
    K.prefix_attention(q, pk, pv, k, v, out, D**-0.5, lens, work[:need])
    assert check() and bool(work[need:].isnan().all())
    last = lens[:, None, None] - L + 1 + torch.arange(L, device=dev)[None, :, None]
    seen = torch.cat((torch.ones(B, L, P, dtype=torch.bool, device=dev), torch.arange(S, device=dev) < last), 2)
    both = [torch.cat((a[None].expand(B, -1, -1, -1), b), 1) for a, b in ((pk, k), (pv, v))]
    o, size, load = reference64(q, *both, D**-0.5, seen)
    assert_near(out.float().cpu().numpy(), o, bound(kind, D**-0.5, o, size, load, both[1].float().abs().max().item(), P + S))


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("L,D", [(1, 64), (40, 128), (128, 96)])
def test_cross_attention_long_tails(dev, kind, L, D):
    """60 000 keys of 2^-16 of the largest's weight, below fp16's normal numbers: they hold 48 % of the weight."""
    K = kern()
    S = 60001
    q = torch.zeros(1, L, 1, D, dtype=TYPES[kind], device=dev)
    k, v = torch.zeros(1, S, 1, D, dtype=TYPES[kind], device=dev), torch.ones(1, S, 1, D, dtype=TYPES[kind], device=dev)
    q[..., 0], k[0, 7, 0, 0], v[0, 7] = 1.0, 16.0, 0.0
    out = torch.empty_like(q)
    K.cross_attention(q, k, v, out, math.log(2), None, None, torch.empty(max(1, K.cross_attention_work(q, k)), device=dev))
    want = 60000 * 2.0**-16 / (1 + 60000 * 2.0**-16)
    # weights are powers of two but for scale's and c's roundings; 60 000 fp32 sums by 16 and by cuts
    assert bool(((out.float() - want).abs() <= want * (HALF[kind] + 60000 / 16 * 2.0**-24 + 2.0**-18)).all())


def test_attentions_share_a_workspace(dev):
    """Calls that run one after another in one stream, with one workspace."""
    K = kern()
    g = torch.Generator(device=dev).manual_seed(9)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g).half()  # noqa: E731
    q, k, v, pk, pv = rnd(4, 40, 4, 64), rnd(4, 3000, 2, 64), rnd(4, 3000, 2, 64), rnd(900, 2, 64), rnd(900, 2, 64)
    need = max(K.cross_attention_work(q, k), K.prefix_attention_work(q, pk, k))
    one = torch.empty(need, device=dev)
    got = [torch.empty_like(q) for _ in range(4)]
    for a, b in ((got[0], got[1]), (got[2], got[3])):
        K.cross_attention(q, k, v, a, 0.125, None, None, one)
        K.prefix_attention(q, pk, pv, k, v, b, 0.125, None, one)
    K.cross_attention(q, k, v, got[0], 0.125, None, None, torch.empty(need, device=dev))
    K.prefix_attention(q, pk, pv, k, v, got[1], 0.125, None, torch.empty(need, device=dev))
    assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3])


def test_registered_ops_take_the_same_calls(dev):
    K = kern()
    ops = K.kernels()
    q, k = torch.randn(2, 3, 4, 64, device=dev).half(), torch.randn(2, 50, 2, 64, device=dev).half()
    a, b = torch.empty_like(q), torch.empty_like(q)
    ops.cross_attention(q, k, k, a, 0.125)
    K.cross_attention(q, k, k, b, 0.125)
    assert torch.equal(a, b)
    ops.prefix_attention(q, k[0], k[1], k, k, a, 0.125)
    K.prefix_attention(q, k[0], k[1], k, k, b, 0.125)
    assert torch.equal(a, b)
    x, g = torch.randn(5, 64, device=dev).half(), torch.ones(64, device=dev)
    h = [torch.empty_like(x) for _ in range(4)]
    ops.residual_norm(x, x, h[0], h[1], 1, g, None, 1, g, None)
    K.residual_norm(x, x, h[2], h[3], 1, g, None, 1, g, None)
    assert torch.equal(h[0], h[2]) and torch.equal(h[1], h[3])


def test_python_refusals_on_the_gpu(dev):
    K = kern()
    q, k = torch.randn(2, 3, 4, 64, device=dev).half(), torch.randn(2, 50, 2, 64, device=dev).half()
    out = torch.empty_like(q)
    bad = [
        (dict(k=k.bfloat16()), "type"), (dict(k=k.cpu()), "device"), (dict(k=k[:1]), "B and D"), (dict(v=k[:, :9]), "one shape"),
        (dict(out=out[:, :2]), "shape"), (dict(out=out.float()), "type"), (dict(q=q[0]), "B, L, heads, D"),
        (dict(q=q.transpose(2, 3).contiguous().transpose(2, 3)), "contiguous columns"),
        (dict(lens=torch.ones(2, device=dev)), "int32"), (dict(lens=torch.ones(3, dtype=torch.int32, device=dev)), "int32"),
        (dict(mask=torch.ones(2, 50, device=dev)), "bool"), (dict(mask=torch.ones(2, 49, dtype=torch.bool, device=dev)), "bool"),
        (dict(mask=torch.ones(50, 2, dtype=torch.bool, device=dev).t()), "contiguous columns"),
        (dict(work=torch.ones(9, device=dev).half()), "fp32"), (dict(out=q), "overlaps"), (dict(scale=0.0), "scale"),
        (dict(q=q.clone().requires_grad_()), "no backward"),
    ]
    for change, word in bad:
        args = dict(q=q.detach(), k=k, v=k, out=out, scale=0.125) | change
        with pytest.raises(RuntimeError, match=word):
            K.cross_attention(**args)
    with pytest.raises(RuntimeError, match=r"\[P, kv_heads, D\]"):
        K.prefix_attention(q.detach(), k[0, :, :1], k[0, :, :1], k, k, out, 0.125)
    x = torch.randn(4, 64, device=dev).half()
    g = torch.ones(64, device=dev)
    for change, word in [(dict(y=x.float()), "type"), (dict(h=None), "h goes"), (dict(gate=g[:8]), "gate"),
                         (dict(gate=torch.ones(3, 64, device=dev)), "multiple of the gate"), (dict(post_gamma=g[:32]), "64 elements"),
                         (dict(gate=torch.ones(0, 64, device=dev)), "gate"), (dict(x=x.t().contiguous().t()), "contiguous rows")]:
        args = dict(x=x, y=x, x_out=torch.empty_like(x), h=torch.empty_like(x), post=1, post_gamma=g, post_beta=None, pre=1,
                    pre_gamma=g, pre_beta=None) | change
        with pytest.raises(RuntimeError, match=word):
            K.residual_norm(**args)


def test_decoder_block_eager_and_captured(dev):
    """A decoder block over an image's tokens: norms, 4-bit linears, head norms with rotation, attention behind the image's tokens
    as a shared prefix, cross attention to another image's tokens, each attention held to the oracle on the inputs it got; the
    captured run replayed over new inputs gives the eager run's bits."""
    K = kern()
    B, L, C, H, KV, P, S = 3, 2, 512, 8, 4, 200, 70
    T, D = B * L, 64
    g = torch.Generator(device=dev).manual_seed(10)
    rnd = lambda *s, std=1.0: torch.randn(*s, device=dev, generator=g) * std  # noqa: E731
    mx = lambda n, c: (torch.empty(n, c // 2, dtype=torch.uint8, device=dev),  # noqa: E731
                       torch.empty(c // 128, n, dtype=torch.int32, device=dev))

    def linear(n):
        codes = mx(n, C)
        K.quant_mx4(rnd(n, C, std=C**-0.5).half(), *codes)
        return codes, rnd(n, std=0.02)

    wide = (H + 2 * KV) * D
    w_qkv, w_o, w_q, w_co = linear(wide), linear(C), linear(H * D), linear(C)
    norms = [(1 + rnd(C, std=0.1), rnd(C, std=0.1)) for _ in range(5)]
    hg = [1 + rnd(D, std=0.1) for _ in range(2)]
    gate = rnd(C, std=0.5)
    ang = torch.arange(400, device=dev)[:, None] * 10000.0 ** (-torch.arange(D // 2, device=dev) / (D // 2))
    cos, sin = ang.cos().contiguous(), ang.sin().contiguous()
    x0, y0 = rnd(T, C).half(), rnd(T, C).half()
    pk, pv = rnd(P, KV, D).half(), rnd(P, KV, D).half()
    cache_k, cache_v = rnd(B, KV, S, D).half().transpose(1, 2), rnd(B, KV, S, D).half().transpose(1, 2)
    enc = rnd(B, 150, 2, KV, D).half()
    mask = torch.rand(B, 150, device=dev, generator=g) < 0.6
    lens = torch.tensor([70, 2, 33], dtype=torch.int32, device=dev)
    positions = (P + lens[:, None] - L + torch.arange(L, device=dev)).flatten().int()

    def block(t):
        """One block into the tensors of t."""
        K.residual_norm(x0, y0, t["x"], t["h"], K.NORM_RMS, norms[0][0], None, K.NORM_LAYER, *norms[1], gate, 0.5)
        K.quant_mx4(t["h"], *t["a"])
        K.gemm_mx4(*t["a"], *w_qkv[0], w_qkv[1], t["qkv"], K.EPI_BIAS_F16)
        rows = t["qkv"].view(T, H + 2 * KV, D)
        q, k, v = rows[:, :H], rows[:, H : H + KV], rows[:, H + KV :]
        K.qk_norm_rope(q, k, q, k, K.NORM_RMS, *hg, None, None, cos, sin, positions)
        at = torch.arange(B, device=dev)[:, None], (lens[:, None] - L + torch.arange(L, device=dev)).long()
        t["k"].copy_(cache_k)
        t["v"].copy_(cache_v)
        t["k"][at], t["v"][at] = k.view(B, L, KV, D), v.view(B, L, KV, D)  # the new tokens' own rows
        K.prefix_attention(q.view(B, L, H, D), pk, pv, t["k"], t["v"], t["o"], D**-0.5, lens, t["work"])
        K.quant_mx4(t["o"].view(T, C), *t["a"])
        K.gemm_mx4(*t["a"], *w_o[0], w_o[1], t["y"], K.EPI_BIAS_F16)
        K.residual_norm(t["x"], t["y"], t["x"], t["h"], K.NORM_RMS, norms[2][0], None, K.NORM_RMS, norms[3][0], None)
        K.quant_mx4(t["h"], *t["a"])
        K.gemm_mx4(*t["a"], *w_q[0], w_q[1], t["q"], K.EPI_BIAS_F16)
        K.cross_attention(t["q"].view(B, L, H, D), enc[:, :, 0], enc[:, :, 1], t["c"], D**-0.5, None, mask, t["work"])
        K.quant_mx4(t["c"].view(T, C), *t["a"])
        K.gemm_mx4(*t["a"], *w_co[0], w_co[1], t["y"], K.EPI_BIAS_F16)
        K.residual_norm(t["x"], t["y"], t["x"], None, K.NORM_LAYER, *norms[4], K.NORM_NONE, None, None, gate)
        return t["x"]

    def tensors():
        e = lambda *s: torch.empty(*s, dtype=torch.float16, device=dev)  # noqa: E731
        t = dict(x=e(T, C), h=e(T, C), y=e(T, C), qkv=e(T, wide), q=e(T, H * D), o=e(B, L, H, D), c=e(B, L, H, D),
                 k=e(B, KV, S, D).transpose(1, 2), v=e(B, KV, S, D).transpose(1, 2), a=mx(T, C))
        need = max(K.prefix_attention_work(t["o"], pk, t["k"]), K.cross_attention_work(t["o"], enc[:, :, 0]))
        return t | dict(work=torch.empty(max(need, 1), device=dev))

    a, b = tensors(), tensors()
    block(a)
    torch.cuda.synchronize()
    assert bool(a["x"].isfinite().all())
    n = lambda t: t.float().cpu().numpy()  # noqa: E731
    q = n(a["qkv"].view(B, L, H + 2 * KV, D)[:, :, :H])
    o, size, load = OC.prefix_attention(q, n(pk), n(pv), n(a["k"]), n(a["v"]), D**-0.5, lens.tolist())
    assert_near(n(a["o"]), o, bound("fp16", D**-0.5, o, size, load, max(np.abs(n(a["v"])).max(), np.abs(n(pv)).max()), P + S))
    o, size, load = OC.cross_attention(n(a["q"].view(B, L, H, D)), n(enc[:, :, 0]), n(enc[:, :, 1]), D**-0.5, None, mask.cpu().numpy())
    assert_near(n(a["c"]), o, bound("fp16", D**-0.5, o, size, load, np.abs(n(enc)).max(), 150))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block(a)
    for _ in range(3):
        x0.copy_(rnd(T, C).half())
        enc.copy_(rnd(*enc.shape).half())
        graph.replay()
        block(b)
        torch.cuda.synchronize()
        assert torch.equal(a["x"], b["x"])
