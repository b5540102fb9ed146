"""Attention to other rows and behind a prefix for scores and values that are not finite, on the GPU, against float64.

Scores are fp32: one of +inf (an infinite element, or a product past fp32's range) makes its row not a number, as the softmax's
inf - inf does; -inf has no weight while another seen key has some. The bar for finite rows is `bound` of the operators' own tests,
for the keys that have a weight.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
from test_cross_attention_gpu import TYPES, assert_near, bound, guarded, kern, reference64

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

INF = math.inf

# B, L, S, H, KV, D by what computes them
CROSS = {
    "streams of eight waves": (2, 3, 700, 4, 2, 64),
    "streams, keys cut": (2, 2, 6000, 4, 2, 128),
    "streams of four waves": (140, 2, 200, 4, 2, 96),
    "two units": (2, 50, 300, 2, 2, 64),
    "two units of groups": (3, 25, 257, 8, 4, 128),
    "tiles": (3, 100, 300, 2, 2, 64),
    "tiles, a streamed rest": (2, 140, 333, 4, 2, 96),
    "tiles, keys cut": (2, 70, 6000, 1, 1, 128),
    "tiles, the last round cut": (9, 1029, 2100, 16, 16, 64),
}
# B, L, P, S, H, KV, D
PREFIX = {
    "streams of both": (1, 4, 300, 40, 8, 4, 64),
    "streams of many sequences": (70, 4, 40, 20, 8, 4, 64),
    "streams of own keys": (5, 2, 1025, 70, 4, 2, 128),
    "two units": (3, 20, 200, 33, 4, 2, 96),
    "tiles": (2, 130, 64, 200, 2, 1, 64),
    "no prefix": (2, 140, 0, 170, 2, 2, 64),
}


def random(dev, kind, seed, *shapes):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(*s, device=dev, generator=g).to(TYPES[kind]) for s in shapes]


def call_cross(dev, kind, q, k, v, scale, lens, mask):
    K = kern()
    out, check = guarded(kind, dev, *q.shape)
    need = K.cross_attention_work(q, k)
    work = torch.full((need + 64,), math.nan, device=dev)
    K.cross_attention(q, k, v, out, scale, lens, mask, work[:need])
    assert check() and bool(work[need:].isnan().all())
    return out


def call_prefix(dev, kind, q, pk, pv, k, v, scale, lens):
    K = kern()
    out, check = guarded(kind, dev, *q.shape)
    need = K.prefix_attention_work(q, pk, k)
    work = torch.full((need + 64,), math.nan, device=dev)
    K.prefix_attention(q, pk, pv, k, v, out, scale, lens, work[:need])
    assert check() and bool(work[need:].isnan().all())
    return out


def own_seen(dev, B, L, S, lens):
    """[B, L, S]: the own keys that a new token sees."""
    n = (torch.full((B,), S, device=dev) if lens is None else lens.clamp(0, S))[:, None, None]
    return torch.arange(S, device=dev) < n - L + 1 + torch.arange(L, device=dev)[:, None]


def assert_rows(kind, got, q, k, v, scale, weighty, bad):
    """weighty [B, L or 1, S]: keys with a finite score; bad [B, L or 1]: rows that are not a number; other rows without keys: 0."""
    B, L = q.shape[:2]
    weighty, bad = weighty.expand(B, L, -1), bad.expand(B, L)
    some = weighty.any(-1)
    got = got.float()
    assert bool(got[bad].isnan().all()), f"{int((~got[bad].isnan()).sum())} finite values in rows that have none"
    assert bool((got[~some & ~bad] == 0).all())
    kept = (weighty & ~bad[..., None]).any(1)[:, :, None, None]  # what no good row needs holds anything
    k, v = k.masked_fill(~kept, 0), v.masked_fill(~kept, 0)
    dummy = weighty | ~some[..., None]
    want = reference64(q.masked_fill(bad[..., None, None], 0), k, v, scale, dummy)
    rows = (some & ~bad).cpu().numpy()
    o, size, load = (x[rows] for x in want)
    if rows.any():
        tol = bound(kind, scale, o, size, load, v.float().abs().max().item(), k.size(1))
        assert_near(got.cpu().numpy()[rows], o, tol)


@pytest.mark.parametrize("kind,how", [("fp16", "key"), ("bf16", "key"), ("fp16", "query"), ("bf16", "query"), ("bf16", "dot"),
                                      ("bf16", "scaled")])
@pytest.mark.parametrize("name", CROSS)
def test_cross_attention_of_an_infinite_score(dev, kind, how, name):
    """An infinity in a key (rows with a negative query there give it no weight) or a query; a dot product past fp32's range, or
    one past it times scale."""
    B, L, S, H, KV, D = CROSS[name]
    q, k0, v = random(dev, kind, 31, (B, L, H, D), (B, S, KV, D), (B, S, KV, D))
    scale = 8.0 if how == "scaled" else D**-0.5
    if how == "scaled":
        q *= 2.0**-6
    turn = (torch.arange(B, device=dev)[:, None] + torch.arange(L, device=dev)) % 3  # 0: infinite scores
    sign = torch.where(turn == 0, 1.0, -1.0).to(q.dtype)[..., None]
    g = torch.Generator(device=dev).manual_seed(32)
    every = torch.ones(B, S, dtype=torch.bool, device=dev)
    for at in (5, 40, S // 2, S - 1):
        k = k0.clone()
        weighty = every.clone()
        if how == "query":
            q[..., 0] = torch.where(turn[..., None] == 0, INF, 0.5).to(q.dtype)
        else:
            size, far = {"key": (1.0, INF), "dot": (2.0**70, 2.0**70), "scaled": (2.0**63, 2.0**63)}[how]
            q[..., 0] = sign * size
            if how != "key":
                k[..., 0] = 0
            k[:, at, :, 0] = far
            weighty[:, at] = False
        assert_rows(kind, call_cross(dev, kind, q, k, v, scale, None, None), q, k, v, scale, weighty[:, None], turn == 0)
        mask = torch.rand(B, S, device=dev, generator=g) < 0.6
        mask[:, at] = True
        got = call_cross(dev, kind, q, k, v, scale, None, mask)
        assert_rows(kind, got, q, k, v, scale, (weighty & mask)[:, None], turn == 0)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("name", PREFIX)
def test_prefix_attention_of_an_infinite_score(dev, kind, name):
    B, L, P, S, H, KV, D = PREFIX[name]
    q, pk0, pv, k0, v = random(dev, kind, 33, (B, L, H, D), (P, KV, D), (P, KV, D), (B, S, KV, D), (B, S, KV, D))
    turn = (torch.arange(B, device=dev)[:, None] + torch.arange(L, device=dev)) % 3
    q[..., 0] = torch.where(turn == 0, 1.0, -1.0).to(q.dtype)[..., None]
    seen = torch.cat((torch.ones(B, L, P, dtype=torch.bool, device=dev), own_seen(dev, B, L, S, None)), 2)
    vs = torch.cat((pv.expand(B, -1, -1, -1), v), 1)
    for at in sorted({*([5, P - 1] if P else []), P, P + S - L, P + S - 1}):
        pk, k = pk0.clone(), k0.clone()
        (pk[at] if at < P else k[:, at - P])[..., 0] = INF
        weighty = seen.clone()
        weighty[:, :, at] = False
        got = call_prefix(dev, kind, q, pk, pv, k, v, D**-0.5, None)
        ks = torch.cat((pk.expand(B, -1, -1, -1), k), 1)
        assert_rows(kind, got, q, ks, vs, D**-0.5, weighty, (turn == 0) & seen[:, :, at])


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("name", CROSS)
def test_cross_attention_of_keys_at_minus_infinity(dev, kind, masked, name):
    """Seen keys whose scores are all -inf are no missing keys: 0 / 0, not 0. With others behind or before them they weigh nothing."""
    B, L, S, H, KV, D = CROSS[name]
    q, k0, v = random(dev, kind, 34, (B, L, H, D), (B, S, KV, D), (B, S, KV, D))
    q[..., 0] = 1.0
    g = torch.Generator(device=dev).manual_seed(35)
    at = torch.arange(S, device=dev)
    lens = torch.full((B,), S, dtype=torch.int32, device=dev)
    lens[0], lens[1] = 0, S - 7  # none in the first
    for gone in (at >= 0, at < S * 7 // 10, at >= 40, at != S - 9):
        minus = gone.expand(B, -1).clone()
        if B > 2:
            minus[2] = False
        k = k0.clone()
        k[..., 0].masked_fill_(minus[..., None], -INF)
        mask, seen = None, at < lens[:, None]
        if masked:
            mask = torch.rand(B, S, device=dev, generator=g) < 0.5
            mask[:, S - 9] = True
            seen = seen & mask
        weighty = seen & ~minus
        bad = seen.any(1) & ~weighty.any(1)
        got = call_cross(dev, kind, q, k, v, D**-0.5, lens, mask)
        assert_rows(kind, got, q, k, v, D**-0.5, weighty[:, None], bad[:, None])


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("name", PREFIX)
def test_prefix_attention_of_keys_at_minus_infinity(dev, kind, name):
    B, L, P, S, H, KV, D = PREFIX[name]
    q, pk0, pv, k0, v = random(dev, kind, 36, (B, L, H, D), (P, KV, D), (P, KV, D), (B, S, KV, D), (B, S, KV, D))
    q[..., 0] = 1.0
    lens = torch.full((B,), S, dtype=torch.int32, device=dev)
    lens[0] = L - 1  # its first token sees the prefix alone, or nothing
    seen = torch.cat((torch.ones(B, L, P, dtype=torch.bool, device=dev), own_seen(dev, B, L, S, lens)), 2)
    vs = torch.cat((pv.expand(B, -1, -1, -1), v), 1)
    at = torch.arange(P + S, device=dev)
    for gone in (at >= 0, at < P, at >= P, at != P + S - L, at >= P + S // 2):
        pk, k = pk0.clone(), k0.clone()
        pk[..., 0].masked_fill_(gone[:P, None], -INF)
        k[..., 0].masked_fill_(gone[P:, None], -INF)
        weighty = seen & ~gone
        bad = seen.any(2) & ~weighty.any(2)
        got = call_prefix(dev, kind, q, pk, pv, k, v, D**-0.5, lens)
        assert_rows(kind, got, q, torch.cat((pk.expand(B, -1, -1, -1), k), 1), vs, D**-0.5, weighty, bad)


# Weights of a row run from 2^8 of its largest score's down (fp16): half a subnormal step, 2^-25, is 2^-33 of the largest.
TAIL = 2.0**-33


@pytest.mark.parametrize("below", [24.625, 25.5, 28.0])
@pytest.mark.parametrize("B,L,D", [(300, 1, 64), (600, 40, 128), (520, 128, 96)])
def test_cross_attention_fp16_tails_below_the_subnormals(dev, below, B, L, D):
    """60 000 keys of 2^-24.6 to 2^-28 of the largest's weight, below the last step of fp16 or just above it, not cut: they hold up
    to 0.2 % of the weight. Weights are exact but for scale's and c's roundings (28 2^-23 in the exponent) and the tails'."""
    S = 60001
    q = torch.zeros(B, L, 1, D, dtype=torch.float16, device=dev)
    k, v = torch.zeros(1, S, 1, D, dtype=torch.float16, device=dev), torch.ones(1, S, 1, D, dtype=torch.float16, device=dev)
    q[..., 0], k[..., 0] = 1.0, -below / 2
    k[0, 7, 0, 0], v[0, 7] = below / 2, 0.0
    assert kern().cross_attention_work(q, k.expand(B, -1, -1, -1)) == 0
    got = call_cross(dev, "fp16", q, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), math.log(2), None, None).float()
    rest = 60000 * 2.0**-below
    want = rest / (1 + rest)
    tol = want * (2.0**-11 + 60000 / 16 * 2.0**-24 + 2.0**-17) + 60000 * TAIL + 2.0**-25
    assert bool(((got - want).abs() <= tol).all()), ((got - want).abs().max().item(), want, tol)


@pytest.mark.parametrize("B,L,D", [(300, 1, 64), (600, 40, 128), (520, 128, 96)])
def test_cross_attention_fp16_tails_of_all_sizes(dev, B, L, D):
    """Scores from the largest's down to 2^-40 of its weight, in no order."""
    S = 40001
    g = torch.Generator(device=dev).manual_seed(37)
    q = torch.zeros(B, L, 1, D, dtype=torch.float16, device=dev)
    k, v = torch.zeros(1, S, 1, D, dtype=torch.float16, device=dev), torch.rand(1, S, 1, D, device=dev, generator=g).half()
    q[..., 0], k[0, :, 0, 0] = 1.0, -torch.linspace(16, 40, S, device=dev)[torch.randperm(S, device=dev, generator=g)].half()
    k[0, 3, 0, 0], v[0, 3] = 0.0, 0.0
    got = call_cross(dev, "fp16", q, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), math.log(2), None, None)
    p = torch.exp2(k[0, :, 0, 0].double())
    want = ((p @ v[0, :, 0].double()) / p.sum()).expand(B, L, 1, D)
    tol = want * (2 * 2.0**-11 + S / 16 * 2.0**-24 + 2.0**-17) + S * TAIL + 2.0**-25
    assert bool(((got.double() - want).abs() <= tol).all()), ((got.double() - want).abs() / tol).max().item()


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("shape", [
    (1, 4, 300, 40, 8, 4, 64), (70, 4, 40, 20, 8, 4, 96), (5, 6, 1025, 70, 4, 2, 128), (3, 20, 200, 33, 4, 2, 96),
    (2, 130, 64, 200, 2, 1, 64), (2, 140, 0, 170, 2, 2, 64), (3, 50, 80, 150, 4, 2, 128), (2, 45, 0, 64, 1, 1, 40),
    (2, 100, 31, 100, 1, 1, 128),
])
def test_prefix_attention_of_values_that_earlier_tokens_do_not_see(dev, kind, shape):
    """Infinities and not-a-numbers in new tokens' values and keys reach the tokens that see them, and no others."""
    B, L, P, S, H, KV, D = shape
    q, pk, pv, k, v = random(dev, kind, 38, (B, L, H, D), (P, KV, D), (P, KV, D), (B, S, KV, D), (B, S, KV, D))
    lens = torch.full((B,), S, dtype=torch.int32, device=dev)
    lens[0] = max(L - 2, 1) if B > 1 else S  # tokens that see the prefix alone, or nothing
    for b in range(B):
        n = int(lens[b])
        v[b, n - 1, :, 0], v[b, n - 1, :, 1], v[b, n - 1, :, 2] = INF, -INF, math.nan
        v[b, n - 1, :, D - 1] = INF
        v[b, n - 2, :, 3], v[b, n - 2, :, 4] = INF, math.nan
        v[b, max(n - 2 * L // 3, 0), :, 5], v[b, n - 1, :, 5] = INF, -INF  # both: not a number
        v[b, max(n - L // 2, 0), :, 6] = -INF
    got = call_prefix(dev, kind, q, pk, pv, k, v, D**-0.5, lens).float()
    seen = torch.cat((torch.ones(B, L, P, dtype=torch.bool, device=dev), own_seen(dev, B, L, S, lens)), 2)
    ks, vs = torch.cat((pk.expand(B, -1, -1, -1), k), 1), torch.cat((pv.expand(B, -1, -1, -1), v), 1)
    # what a row sees that is not finite, by column; every weight is far above 0
    some = seen.any(-1, keepdim=True)
    o, size, load = reference64(q, ks, vs.masked_fill(~vs.isfinite(), 0), D**-0.5, seen | ~some)
    G = H // KV
    hits = [(seen.float() @ f.float().reshape(B, P + S, KV * D)).view(B, L, KV, D).repeat_interleave(G, 2) > 0
            for f in (vs == INF, vs == -INF, vs.isnan())]
    bad = hits[2] | (hits[0] & hits[1])
    assert bool(got[bad].isnan().all())
    assert bool((got[hits[0] & ~bad] == INF).all() and (got[hits[1] & ~bad] == -INF).all())
    plain = ~(bad | hits[0] | hits[1])
    assert bool((got[plain & ~some[..., None]] == 0).all())
    at = (plain & some[..., None]).cpu().numpy()
    tol = bound(kind, D**-0.5, o, size, load, vs[vs.isfinite()].float().abs().max().item(), P + S)
    assert_near(got.cpu().numpy()[at], o[at], np.broadcast_to(tol, o.shape)[at])
    # a key that is not a number: the tokens that see it, and no others
    v = v.masked_fill(~v.isfinite(), 0)
    for b in range(B):
        k[b, int(lens[b]) - 1] = math.nan
    got = call_prefix(dev, kind, q, pk, pv, k, v, D**-0.5, lens).float()
    last = torch.zeros(B, L, dtype=torch.bool, device=dev)
    last[:, -1] = True
    assert bool(got[last].isnan().all() and got[~last].isfinite().all())


@pytest.mark.parametrize("kind,D", [("fp16", 48), ("bf16", 96), ("fp16", 128), ("bf16", 64)])
@pytest.mark.parametrize("with_lens", [False, True])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("B,L,H,KV", [(280, 1, 4, 1), (70, 5, 24, 4)])
def test_cross_attention_streams_of_four_waves(dev, kind, D, with_lens, masked, B, L, H, KV):
    """More sequences and key heads than CUs, up to 32 rows of each: four waves a workgroup, keys uncut."""
    S = 333
    q, k, v = random(dev, kind, 39, (B, L, H, D), (B, S, KV, D), (B, S, KV, D))
    assert B * KV > 256 and kern().cross_attention_work(q, k) == 0
    g = torch.Generator(device=dev).manual_seed(40)
    lens = mask = None
    seen = torch.ones(B, S, dtype=torch.bool, device=dev)
    if with_lens:
        lens = torch.randint(0, S + 1, (B,), device=dev, generator=g).int()
        lens[:6] = torch.tensor([0, 1, 32, 33, S + 5, -3], device=dev)
        seen = torch.arange(S, device=dev) < lens[:, None]
    if masked:
        mask = torch.rand(B, S, device=dev, generator=g) < torch.linspace(0.02, 0.98, B, device=dev)[:, None]
        mask[3], mask[7], mask[8, :] = False, True, torch.arange(S, device=dev) == S - 1
        seen = seen & mask
    k[~seen], v[~seen] = math.nan, math.nan
    got = call_cross(dev, kind, q, k, v, D**-0.5, lens, mask)
    assert_rows(kind, got, q, k, v, D**-0.5, seen[:, None], torch.zeros(B, 1, dtype=torch.bool, device=dev))


def test_cross_attention_of_more_rows_than_a_join_takes(dev):
    """67 million rows, of which the last round's are cut and joined: that round's head and sequence, and rows of all others."""
    B, L, S, H, D = 8, 524544, 2100, 16, 8
    q, k, v = random(dev, "fp16", 42, (1, L, H, D), (B, S, H, D), (B, S, H, D))
    out = call_cross(dev, "fp16", q.expand(B, -1, -1, -1), k, v, D**-0.5, None, None)
    every = torch.ones(1, 1, S, dtype=torch.bool, device=dev)
    for b, h, rows in [(B - 1, H - 1, slice(L - 40000, L)), (B - 1, H - 1, slice(0, 1000))] + [
            (b, h, slice(b * 65536 + h * 64, None, 99991)) for b in range(B) for h in range(H)]:
        args = q[:, rows, h : h + 1], k[b : b + 1, :, h : h + 1], v[b : b + 1, :, h : h + 1]
        o, size, load = reference64(*args, D**-0.5, every)
        got = out[b : b + 1, rows, h : h + 1].float().cpu().numpy()
        assert_near(got, o, bound("fp16", D**-0.5, o, size, load, args[2].float().abs().max().item(), S))
