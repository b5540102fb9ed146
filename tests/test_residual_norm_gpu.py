"""The residual stream between two norms on the GPU, against the float64 oracle.

Bar: u half a step of the type for either output, plus fp32 roundings. A mean or a sum of squares takes at most 64 of them
in a row (32 columns a lane, the lanes, the waves), 2^-18 relative to the mean of the absolute values; a normed value is then off by
2^-17 of what it is made of. The error of the sum s = x + scale gate N(y) goes through the second norm at most twice, times
gamma / sigma, as itself and through the mean and sigma.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import cross_attention as OC

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
HALF = {"fp16": 2.0**-11, "bf16": 2.0**-8}
TINY = {"fp16": 2.0**-25, "bf16": 2.0**-133}


def kern():
    from foidfinder_amd import kernels as K

    return K


def normed_error(x, kind, gamma, beta, eps, err_in):
    """Bound of |fp32 norm(x~) - norm(x)| for inputs within err_in of x."""
    if kind == 0:
        return err_in
    centre = x.mean(-1, keepdims=True) if kind == 2 else np.zeros((x.shape[0], 1))
    r = 1.0 / np.sqrt(((x - centre) ** 2).mean(-1, keepdims=True) + eps)
    g = np.abs(gamma)
    out = np.abs(x - centre) * r * g
    lost = np.abs(x).mean(-1, keepdims=True) * r * g if kind == 2 else 0.0
    through = err_in.max(-1, keepdims=True) * r * (2 * g + 2 * out)
    return 2.0**-17 * (out + lost) + (2.0**-22 * np.abs(beta) if kind == 2 else 0.0) + through


def run(dev, kind, T, C, post, pre, gate=None, *, scale=1.0, eps=1e-6, seed=0, gate_type=None, pad=0, place="new", x=None, y=None):
    """gate: rows of the gate or None; pad: elements between rows; place: where the outputs go."""
    K = kern()
    rng = np.random.default_rng(seed)
    dt = TYPES[kind]

    def rows(a):
        wide = torch.full((T, C + pad), 3.0, dtype=dt, device=dev)
        wide[:, :C] = torch.from_numpy(a.astype(np.float32)).to(dev)
        return wide, wide[:, :C]

    xn = rng.standard_normal((T, C)) if x is None else x
    if x is None:
        xn[:, rng.integers(C)] *= 30.0
    xw, xt = rows(xn)
    yw, yt = rows(rng.standard_normal((T, C)) * 0.7 + 0.3 if y is None else y)
    xn, yn = xt.float().cpu().numpy(), yt.float().cpu().numpy()
    par = {}
    for name, n in (("post", post), ("pre", pre)):
        g = (1 + 0.2 * rng.standard_normal(C)).astype(np.float32) if n else None
        b = (0.2 * rng.standard_normal(C)).astype(np.float32) if n == 2 else None
        par[name] = (g, b), tuple(None if p is None else torch.from_numpy(p).to(dev) for p in (g, b))
    gt = gn = None
    if gate is not None:
        gt = torch.from_numpy(rng.standard_normal((gate, C)).astype(np.float32)).to(dev).to(gate_type or dt)
        gn = gt.float().cpu().numpy()
    if place == "new":
        (ow, xo), (hw, h) = rows(np.full((T, C), 9.0)), rows(np.full((T, C), 9.0))
    elif place == "same":
        (ow, xo), (hw, h) = (xw, xt), (yw, yt)
    else:
        (ow, xo), (hw, h) = (yw, yt), (xw, xt)
    K.residual_norm(xt, yt, xo, h if pre else None, post, *par["post"][1], pre, *par["pre"][1], gt, scale, eps)
    torch.cuda.synchronize()
    assert bool((ow[:, C:] == 3).all() and (hw[:, C:] == 3).all()), "wrote between the rows"
    (pg, pb), (qg, qb) = par["post"][0], par["pre"][0]
    s, want = OC.residual_norm(xn, yn, post, pg, pb, pre, qg, qb, gn, scale, eps)
    factor = np.abs(scale) * (1.0 if gn is None else np.abs(np.repeat(gn, T // gate, 0)).astype(np.float64))
    z = OC.norm(yn.astype(np.float64), post, pg, pb, eps)
    ez = normed_error(yn.astype(np.float64), post, pg, pb, eps, np.zeros((T, C)))
    es = factor * (ez + 2.0**-22 * np.abs(z)) + 2.0**-23 * np.abs(s)
    u, tiny = HALF[kind], TINY[kind]
    err = np.abs(xo.float().cpu().numpy() - s)
    assert (err <= u * np.abs(s) + 2 * es + tiny).all(), (err - u * np.abs(s) - 2 * es).max()
    if pre:
        eh = normed_error(s, pre, qg, qb, eps, es)
        err = np.abs(h.float().cpu().numpy() - want)
        assert (err <= u * np.abs(want) + 2 * eh + tiny).all(), (err - u * np.abs(want) - 2 * eh).max()


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("C", [8, 64, 128, 136, 256, 264, 512, 520, 1024, 1032, 1280, 2048, 2056, 4096, 4104, 8192, 8200, 16384])
def test_residual_norm_widths(dev, kind, C):
    for n, (post, pre) in enumerate([(1, 1), (2, 2), (0, 2), (1, 0)]):
        run(dev, kind, 5, C, post, pre, seed=n)


@pytest.mark.parametrize("post", [0, 1, 2])
@pytest.mark.parametrize("pre", [0, 1, 2])
def test_residual_norm_norms_and_gates(dev, post, pre):
    for n, (gate, t) in enumerate([(None, None), (1, None), (6, None), (12, None), (1, torch.float32), (4, torch.float32)]):
        run(dev, "fp16" if n % 2 else "bf16", 12, 400, post, pre, gate, gate_type=t, scale=0.5, seed=n, pad=16)


@pytest.mark.parametrize("T,C", [(1, 1024), (3, 96), (700, 512), (5000, 200), (3001, 1024), (1500, 4096), (901, 2304)])
def test_residual_norm_rows(dev, T, C):
    """One row, and more rows than the resident workgroups hold at once."""
    run(dev, "bf16", T, C, 2, 1, T)
    run(dev, "fp16", T, C, 1, 2, 1, pad=8)


@pytest.mark.parametrize("place", ["same", "crossed"])
@pytest.mark.parametrize("C", [72, 1024, 2600])
def test_residual_norm_in_place(dev, place, C):
    run(dev, "fp16", 2000, C, 2, 2, 1, place=place)
    run(dev, "bf16", 3, C, 1, 1, None, place=place, pad=8)


@pytest.mark.parametrize("C", [256, 3000])
def test_residual_norm_of_equal_zero_and_far_rows(dev, C):
    rng = np.random.default_rng(0)
    equal, zero = np.full((4, C), 5.0), np.zeros((4, C))
    run(dev, "fp16", 4, C, 2, 2, x=zero, y=equal, eps=1e-5)  # no variance: the betas alone
    run(dev, "fp16", 4, C, 1, 1, x=zero, y=zero, eps=1e-5)
    run(dev, "bf16", 4, C, 2, 2, x=zero, y=200.0 + rng.standard_normal((4, C)))  # a mean far from 0
    run(dev, "bf16", 4, C, 1, 1, x=zero, y=1e-20 * rng.standard_normal((4, C)), eps=1e-38)  # a subnormal eps and mean square


def test_residual_norm_keeps_what_is_not_finite_in_its_row(dev):
    K = kern()
    x = torch.randn(9, 1536, device=dev).half()
    y = torch.randn(9, 1536, device=dev).half()
    g = torch.ones(1536, device=dev)
    y[4, 7], x[6, 1535] = float("nan"), float("inf")
    xo, h = torch.empty_like(x), torch.empty_like(x)
    K.residual_norm(x, y, xo, h, 1, g, None, 1, g, None)
    rows = torch.arange(9, device=dev)
    assert bool(xo[4].isnan().all() and h[4].isnan().all() and xo[6, 1535].isinf() and h[6, 1535].isnan())
    assert bool(xo[(rows != 4) & (rows != 6)].isfinite().all() and h[(rows != 4) & (rows != 6)].isfinite().all())


def test_residual_norm_of_no_rows(dev):
    x = torch.empty(0, 64, device=dev).half()
    g = torch.ones(64, device=dev)
    kern().residual_norm(x, x.clone(), x.clone(), x.clone(), 1, g, None, 1, g, None)


def test_residual_norm_on_streams_and_in_graphs(dev):
    K = kern()
    x, y = torch.randn(300, 2304, device=dev).half(), torch.randn(300, 2304, device=dev).half()
    g, b = torch.randn(2304, device=dev), torch.randn(2304, device=dev)
    a, c = [torch.empty_like(x) for _ in range(2)], [torch.empty_like(x) for _ in range(2)]
    call = lambda o: K.residual_norm(x, y, o[0], o[1], 2, g, b, 2, b, g, g, 0.5)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(a)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(a)
    for _ in range(4):
        x.copy_(torch.randn_like(x))
        y.copy_(torch.randn_like(y))
        graph.replay()
        call(c)
        torch.cuda.synchronize()
        assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


@pytest.mark.parametrize("kind,value", [("fp16", 300.0), ("fp16", -60000.0), ("fp16", 0.1), ("bf16", 300.0), ("bf16", 1e30)])
@pytest.mark.parametrize("C", [8, 72, 200, 1000, 1032, 3000, 5000, 8184])
def test_residual_norm_of_constant_rows(dev, kind, value, C):
    """Equal elements have no variance: LayerNorm leaves beta. Their sum has at most 11 + 13 significant bits, as fp32 holds, so that
    the mean is exact."""
    K = kern()
    dt = TYPES[kind]
    x = torch.full((3, C), value, device=dev).to(dt)
    zero = torch.zeros_like(x)
    g = torch.Generator(device=dev).manual_seed(41)
    gamma, beta = 1 + 0.2 * torch.randn(C, device=dev, generator=g), torch.randn(C, device=dev, generator=g)
    xo, h = torch.empty_like(x), torch.empty_like(x)
    K.residual_norm(zero, x, xo, None, K.NORM_LAYER, gamma, beta, K.NORM_NONE, None, None)
    assert torch.equal(xo, beta.to(dt).expand(3, -1))
    K.residual_norm(x, zero, xo, h, K.NORM_NONE, None, None, K.NORM_LAYER, gamma, beta)
    assert torch.equal(xo, x) and torch.equal(h, beta.to(dt).expand(3, -1))
