"""GPU: nirrt_star_amd.nnops against plain 64-bit evaluations.

Tolerances are bounds, element by element, from the arithmetic the kernels state: a sum of n products in fp32 is off by at most
(n + 2) 2^-24 sum |a b|; a rounding to the element type by half a step (eps / 2 of the value, 2^-25 below f16's normals); exp, erfc and the
quotient of an activation by a few 2^-24; dz and g are rounded to the element type before their products; p = exp(l - lse)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half(dt):
    return torch.finfo(dt).eps / 2


def floor_of(dt):
    """half a step of the smallest numbers"""
    return 2.0 ** -25 if dt == torch.float16 else 1e-38


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, g, dt, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt)


def act64(z, name):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "gelu": lambda: z * torch.special.ndtr(z), "silu": lambda: z * torch.sigmoid(z)}[name]()


def slope64(z, name):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).double()
    if name == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))


def within(got, want, bound, dt):
    got = got.double()
    tol = bound + half(dt) * (want.abs() + bound) + floor_of(dt)
    bad = ~((got - want).abs() <= tol)
    assert got.shape == want.shape and not bad.any(), "%d of %d beyond the bound, worst %.3g of it" % (
        int(bad.sum()), bad.numel(), float(((got - want).abs() / tol).max()))


def linear64(x, w, b, r, act):
    x, w = x.double(), w.double()
    k = w.shape[1]
    z, s = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, s = z + b.double(), s + b.double().abs()
    ez = (k + 2) * U * s
    y = act64(z, act)
    ey = 1.2 * ez + (16 * U * (1 + z.abs()) if act in ("gelu", "silu") else 0)      # slopes are below 1.13
    if r is not None:
        y = y + r.double()
        ey = ey + U * y.abs()
    return z, ez, y, ey


SHAPES = [(1, 1, 1), (1, 128, 128), (3, 5, 2), (7, 515, 321), (31, 16, 1000), (64, 64, 64), (130, 96, 36), (257, 33, 70), (300, 8, 129),
          (1000, 260, 132), (8, 4096, 64), (2, 3000, 3)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_forward(m, k, n, act, dt):
    from nirrt_star_amd import nnops
    g = gen(m * 7 + k + n)
    x, w, b, r = randn((m, k), g, dt), randn((n, k), g, dt, k ** -0.5), randn((n,), g, dt), randn((m, n), g, dt)
    for bias, res in ((None, None), (b, r), (b, None)):
        _, _, y, ey = linear64(x, w, bias, res, act)
        within(nnops.linear_act(x, w, bias, res, activation=act), y, ey, dt)


@pytest.mark.parametrize("dt", TYPES)
def test_linear_layouts(dt):
    """rows with padding, rows off 16 bytes, a transposed weight, more dimensions, an expanded input, an overlapping one"""
    from nirrt_star_amd import nnops
    g = gen(5)
    wide, w, b = randn((90, 200), g, dt), randn((40, 72), g, dt, 0.1), randn((41,), g, dt)[1:]
    wt = randn((72, 40), g, dt, 0.1).t()
    flat = randn((4000,), g, dt)
    for x in (wide[:, 8:80], wide[:, 3:75], wide[::3, 1:73], wide[:1, 5:77], wide[:, ::2][:, :72], wide[5, 2:74].expand(6, 72),
              flat.as_strided((30, 72), (50, 1)), wide[:, 0:72].reshape(3, 30, 72), wide[0, 4:76]):
        for ww in (w, wt, randn((40, 73), g, dt, 0.1)[:, 1:]):
            r = randn(x.shape[:-1] + (43,), g, dt)[..., 2:42]
            _, _, y, ey = linear64(x, ww, b, r, "silu")
            within(nnops.linear_act(x, ww, b, r, activation="silu"), y, ey, dt)


def test_linear_empty_and_special_values():
    from nirrt_star_amd import nnops
    w, b = torch.randn(5, 4, device="cuda"), torch.randn(5, device="cuda")
    assert nnops.linear_act(torch.zeros(0, 4, device="cuda"), w, b).shape == (0, 5)
    assert nnops.linear_act(torch.zeros(2, 0, 4, device="cuda"), w, b, activation="relu").shape == (2, 0, 5)
    assert nnops.linear_act(torch.zeros(3, 4, device="cuda"), w[:0]).shape == (3, 0)
    y = nnops.linear_act(torch.zeros(3, 0, device="cuda"), w[:, :0], b, activation="relu")        # no inputs: act(b)
    assert torch.equal(y, b.clamp(min=0).expand(3, 5))
    x = torch.randn(70, 4, device="cuda")
    x[3, 1], x[9, 0], x[20, 2] = float("nan"), float("inf"), float("-inf")
    for act in ("none", "relu", "gelu", "silu"):
        y = nnops.linear_act(x, w, b, activation=act)
        rows = torch.ones(70, dtype=torch.bool)
        rows[[3, 9, 20]] = False
        assert torch.isnan(y[3]).all() and torch.isfinite(y[rows.cuda()]).all()
        assert not torch.isfinite(y[9]).any() or act != "none"
    # empty tensors through the backward pass
    for m, n, k in ((0, 5, 4), (3, 0, 4), (3, 5, 0)):
        leaves = [torch.randn(s, device="cuda", requires_grad=True) for s in ((m, k), (n, k), (n,))]
        y = nnops.linear_act(leaves[0], leaves[1], leaves[2], activation="silu")
        got = torch.autograd.grad(y.sum(), leaves)
        assert [tuple(t.shape) for t in got] == [(m, k), (n, k), (n,)] and all(bool((t == 0).all()) for t in got[:2])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
@pytest.mark.parametrize("m,k,n", [(1, 128, 128), (7, 515, 321), (130, 96, 36), (257, 33, 70), (2000, 260, 132), (5000, 16, 8), (3, 1, 2)])
def test_linear_gradients(m, k, n, act, dt, dy=None):
    from nirrt_star_amd import nnops
    g = gen(m + k * 3 + n)
    x, w, b, r = randn((m, k), g, dt), randn((n, k), g, dt, k ** -0.5), randn((n,), g, dt), randn((m, n), g, dt)
    dy = randn((m, n), g, dt) if dy is None else dy
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    y = nnops.linear_act(*leaves, activation=act)
    dx, dw, db, dr = torch.autograd.grad(y, leaves, dy)
    z, ez, y64, ey = linear64(x, w, b, r, act)
    within(y, y64, ey, dt)
    assert torch.equal(dr, dy)
    dy64 = dy.double()
    dz = dy64 * slope64(z, act)
    # z is kept in the element type; act'' is below 0.8
    edz = dy64.abs() * (0.8 * (ez + half(dt) * (z.abs() + ez) + floor_of(dt)) + 16 * U * (1 + z.abs())) if act != "none" else torch.zeros_like(dz)
    within(db, dz.sum(0), edz.sum(0) + (m + 2) * U * (dz.abs() + edz).sum(0), dt)
    if act != "none":
        edz = edz + half(dt) * (dz.abs() + edz) + floor_of(dt)
    top = dz.abs() + edz
    within(dx, dz @ w.double(), edz @ w.double().abs() + (n + 2) * U * (top @ w.double().abs()), dt)
    within(dw, dz.t() @ x.double(), edz.t() @ x.double().abs() + (m + 2) * U * (top.t() @ x.double().abs()), dt)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("with_res", [False, True])
def test_linear_relu_gradients_are_exact_on_whole_numbers(dt, with_res):
    """small whole numbers: every sum is exact, z (a half more) is never 0 and keeps its sign in the element type"""
    from nirrt_star_amd import nnops
    g = gen(11)
    m, k, n = 150, 12, 35
    ints = lambda s, hi: torch.randint(-hi, hi + 1, s, generator=g, device="cuda").to(dt)
    x, w, dy, r = ints((m, k), 2), ints((n, k), 1), ints((m, n), 1), ints((m, n), 2)
    b = ints((n,), 3) + 0.5
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = nnops.linear_act(*leaves, residual=r if with_res else None, activation="relu")
    got = torch.autograd.grad(y, leaves, dy)
    z = x.double() @ w.double().t() + b.double()
    dz = dy.double() * (z > 0)
    assert torch.equal(y.double(), z.clamp(min=0) + (r.double() if with_res else 0))
    for a, e in zip(got, (dz @ w.double(), dz.t() @ x.double(), dz.sum(0))):
        assert torch.equal(a, e.to(dt))


def test_linear_gradients_against_differences():
    from nirrt_star_amd import nnops
    g = gen(2)
    for act in ("gelu", "silu"):
        x, w, b = (randn(s, g, torch.float32) for s in ((5, 6), (4, 6), (4,)))
        dy = randn((5, 4), g, torch.float32)
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        grads = torch.autograd.grad(nnops.linear_act(*leaves, activation=act), leaves, dy)
        for i, t in enumerate((x, w, b)):
            d = torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64)
            f = lambda h: (act64((x.double() + (h * d if i == 0 else 0)) @ (w.double() + (h * d if i == 1 else 0)).t()
                                 + b.double() + (h * d if i == 2 else 0), act) * dy.double()).sum()
            slope = float(f(1e-5) - f(-1e-5)) / 2e-5
            scale = float((grads[i].double().abs() * d.abs()).sum())
            assert abs(slope - float((grads[i].double() * d).sum())) <= 100 * U * scale + 1e-7 * scale


def test_linear_wants_only_what_is_asked():
    from nirrt_star_amd import nnops
    x = torch.randn(9, 8, device="cuda")
    w = torch.randn(6, 8, device="cuda", requires_grad=True)
    r = torch.randn(9, 6, device="cuda", requires_grad=True)
    y = nnops.linear_act(x, w, None, r, activation="silu")
    gw, gr = torch.autograd.grad(y.sum(), [w, r])            # (dy is an expanded scalar)
    assert gw.shape == (6, 8) and torch.equal(gr, torch.ones_like(r))
    assert not nnops.linear_act(x, w.detach(), activation="relu").requires_grad
    y = nnops.linear_act(x, w.detach(), None, r, activation="gelu")     # only the residual
    assert torch.equal(torch.autograd.grad(y.sum(), r)[0], torch.ones_like(r))
    dy = torch.ones(9, 6, device="cuda", requires_grad=True)
    h, = torch.autograd.grad(nnops.linear_act(x, w), w, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):       # differentiable once
        h.sum().backward()


def test_linear_refusals():
    from nirrt_star_amd import nnops
    x, w = torch.zeros(3, 4, device="cuda"), torch.zeros(5, 4, device="cuda")
    for call in (lambda: nnops.linear_act(x, w[:, :3]), lambda: nnops.linear_act(x, w.half()), lambda: nnops.linear_act(x.double(), w.double()),
                 lambda: nnops.linear_act(x, w, torch.zeros(4, device="cuda")), lambda: nnops.linear_act(x, w, residual=torch.zeros(3, 4, device="cuda")),
                 lambda: nnops.linear_act(x, w, residual=torch.zeros(5, device="cuda")), lambda: nnops.linear_act(x, w.cpu()),
                 lambda: nnops.linear_act(x, w[0]), lambda: nnops.linear_act(x.to(torch.int32), w)):
        with pytest.raises(ValueError):
            call()


# ---- cross entropy ---------------------------------------------------------------------------------------------------------------------
def ce64(x, w, b, t, cw, ignore):
    x, w = x.double(), w.double()
    v, k = w.shape
    l, s = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        l, s = l + b.double(), s + b.double().abs()
    el = (k + 2) * U * s
    lse = torch.logsumexp(l, 1)
    keep = t != ignore
    ts = torch.where(keep, t, torch.zeros_like(t))
    wt = torch.where(keep, cw.double()[ts] if cw is not None else torch.ones_like(lse), torch.zeros_like(lse))
    # the running sum: at most v / 4 + 64 terms in a lane and 32 joins, each exp good to 8 2^-24 and 3 |argument| 2^-24 (arguments that
    # count are above -88); max and log add theirs
    elist = el.max(1)[0] + (v / 4 + 96 + 8) * U + 8 * U * (1 + lse.abs())
    lt = l.gather(1, ts[:, None]).squeeze(1)
    nll = torch.where(keep, wt * (lse - lt), torch.zeros_like(lse))
    enll = wt * (elist + el.gather(1, ts[:, None]).squeeze(1) + 4 * U * (lse.abs() + lt.abs()))
    return l, el, lse, elist, wt, ts, keep, nll, enll


CE_SHAPES = [(1, 1, 2), (1, 128, 1), (5, 3, 7), (40, 128, 2), (64, 64, 64), (129, 33, 17), (300, 100, 1000), (513, 260, 130), (2, 16, 5000), (1000, 8, 33)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,k,v", CE_SHAPES)
@pytest.mark.parametrize("reduction,weighted,bias", [("mean", True, True), ("sum", False, False), ("none", True, False), ("mean", False, True)])
def test_cross_entropy(rows, k, v, reduction, weighted, bias, dt):
    from nirrt_star_amd import nnops
    g = gen(rows + 5 * k + v)
    x, w = randn((rows, k), g, dt), randn((v, k), g, dt, 1.5 * k ** -0.5)
    b = randn((v,), g, dt) if bias else None
    cw = torch.rand(v, generator=g, device="cuda") * 3 + 0.1 if weighted else None
    t = torch.randint(0, v, (rows,), generator=g, device="cuda")
    t = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.2, torch.full_like(t, -100), t)
    t[0] = v - 1
    leaves = [q.clone().requires_grad_(True) for q in (x, w) + ((b,) if bias else ())]
    loss = nnops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2] if bias else None, class_weight=cw, reduction=reduction)
    l, el, lse, elist, wt, ts, keep, nll, enll = ce64(x, w, b, t, cw, -100)
    assert loss.dtype == torch.float32
    if reduction == "none":
        within(loss, nll, enll, torch.float32)
        dloss = torch.randn(rows, generator=g, device="cuda")
        coef = dloss.double() * wt
    else:
        div = wt.sum() if reduction == "mean" else torch.ones_like(wt.sum())
        within(loss, nll.sum() / div, (enll.sum() + 4 * U * nll.sum()) / div, torch.float32)
        dloss = torch.tensor(1.5, device="cuda")
        coef = 1.5 * wt / div
    got = torch.autograd.grad(loss, leaves, dloss)
    p = torch.exp(l - lse[:, None])
    ep = p * (el + elist[:, None] + 4 * U * ((l - lse[:, None]).abs() + 4)) * 1.01
    one = torch.zeros_like(p).scatter_(1, ts[:, None], 1.0)
    c = coef[:, None]
    gm = c * (p - one)
    eg = c.abs() * (ep + 8 * U * (p + one))
    # rounded to the element type relative to the largest coefficient (f16: lifted by 4096)
    eg = eg + half(dt) * (gm.abs() + eg) + floor_of(dt) / (4096 if dt == torch.float16 else 1) * coef.abs().max()
    eg[~keep] = 0
    top = gm.abs() + eg
    wa, xa = w.double().abs(), x.double().abs()
    within(got[0], gm @ w.double(), eg @ wa + (v + 4) * U * (top @ wa), dt)
    within(got[1], gm.t() @ x.double(), eg.t() @ xa + (rows + 4) * U * (top.t() @ xa), dt)
    if bias:
        within(got[2], gm.sum(0), eg.sum(0) + (rows + 4) * U * top.sum(0), dt)
    assert (got[0][~keep] == 0).all()


def test_cross_entropy_ignored_rows_masked_classes_and_bad_targets():
    from nirrt_star_amd import nnops
    g = gen(3)
    rows, k, v = 70, 24, 19
    x, w, b = randn((rows, k), g, torch.float32), randn((v, k), g, torch.float32), randn((v,), g, torch.float32)
    t = torch.randint(0, v, (rows,), generator=g, device="cuda")
    # what an ignored row holds does not matter, NaN included
    t2, x2 = t.clone(), x.clone()
    t2[5:20] = 255
    x2[5:20] = float("nan")
    leaves = [q.clone().requires_grad_(True) for q in (x2, w, b)]
    loss = nnops.linear_cross_entropy(leaves[0], leaves[1], t2, bias=leaves[2], ignore_index=255)
    got = torch.autograd.grad(loss, leaves)
    rest = torch.cat([torch.arange(5), torch.arange(20, rows)]).cuda()
    l64 = [q.double().requires_grad_(True) for q in (x[rest], w, b)]
    want = torch.nn.functional.cross_entropy(l64[0] @ l64[1].t() + l64[2], t[rest])
    wg = torch.autograd.grad(want, l64)
    assert abs(float(loss) - float(want)) < 1e-5 and (got[0][5:20] == 0).all()
    for a, e in ((got[0][rest], wg[0]), (got[1], wg[1]), (got[2], wg[2])):
        assert torch.isfinite(a).all() and (a.double() - e).abs().max() < 1e-5 * max(1.0, float(e.abs().max()))
    # classes masked by -inf: probability and gradient zero
    bm = b.clone()
    bm[3:9] = float("-inf")
    t3 = torch.where((t >= 3) & (t < 9), torch.zeros_like(t), t)
    leaves = [q.clone().requires_grad_(True) for q in (x, w, bm)]
    loss = nnops.linear_cross_entropy(leaves[0], leaves[1], t3, bias=leaves[2])
    got = torch.autograd.grad(loss, leaves)
    assert torch.isfinite(loss) and all(torch.isfinite(q).all() for q in got) and (got[1][3:9] == 0).all() and (got[2][3:9] == 0).all()
    # the type's lowest value as a mask: the same
    bl = b.clone()
    bl[3:9] = torch.finfo(torch.float32).min
    low = nnops.linear_cross_entropy(x, w, t3, bias=bl)
    assert torch.equal(low, loss.detach())
    # every class masked: no distribution
    assert torch.isnan(nnops.linear_cross_entropy(x, w, t, bias=torch.full_like(b, float("-inf"))))
    # no row counts
    none = torch.full_like(t, -100)
    assert torch.isnan(nnops.linear_cross_entropy(x, w, none, bias=b)) and float(nnops.linear_cross_entropy(x, w, none, bias=b, reduction="sum")) == 0.0
    leaf = w.clone().requires_grad_(True)
    gw, = torch.autograd.grad(nnops.linear_cross_entropy(x, leaf, none, bias=b, reduction="sum"), leaf)
    assert (gw == 0).all()
    # a target that is no class
    for bad in (v, -1):
        tb = t.clone()
        tb[7] = bad
        per = nnops.linear_cross_entropy(x, w, tb, bias=b, reduction="none")
        assert torch.isnan(per[7]) and torch.isfinite(per[:7]).all() and torch.isfinite(per[8:]).all()
        assert torch.isnan(nnops.linear_cross_entropy(x, w, tb, bias=b))
    # no rows, no features
    assert float(nnops.linear_cross_entropy(x[:0], w, t[:0], reduction="sum")) == 0.0
    per = nnops.linear_cross_entropy(x[:, :0], w[:, :0], t, bias=b, reduction="none")
    assert (per.double() - torch.nn.functional.cross_entropy(b.double().expand(rows, v), t, reduction="none")).abs().max() < 1e-5
    # large scores do not overflow
    assert torch.isfinite(nnops.linear_cross_entropy(x * 1e4, w, t, bias=b))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [5, 19])
def test_cross_entropy_masks_of_the_lowest_value(v, dt):
    """a masked target (a loss near the largest number, not infinite) and a row with nothing but masked classes (as good as equal scores)"""
    from nirrt_star_amd import nnops
    g = gen(v)
    rows, k, low = 66, 40, torch.finfo(dt).min
    x, w, b = randn((rows, k), g, dt), randn((v, k), g, dt, k ** -0.5), randn((v,), g, dt)
    t = torch.randint(0, v - 1, (rows,), generator=g, device="cuda")
    t[3] = v - 1
    b[v - 1] = low
    per = nnops.linear_cross_entropy(x, w, t, bias=b, reduction="none")
    assert torch.isfinite(per).all() and abs(float(per[3]) + low) <= 4 * U * abs(low)
    for bias in (b, torch.full_like(b, low)):
        leaves = [q.clone().requires_grad_(True) for q in (x, w, bias)]
        loss = nnops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2], reduction="none")
        got = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
        # (scores 3e38 apart leave nothing of the others; 64 bits hold them to 4e22, so equal ones are equal there too)
        p = torch.softmax(x.double() @ w.double().t() + bias.double(), 1)
        one = torch.zeros_like(p).scatter_(1, t[:, None], 1.0)
        gm = p - one
        # scores to (k + 3) 2^-24 sum |x w| absolutely, exponentials and sums a few 2^-24; gm is rounded to the element type
        eg = ((k + 3) * U * 2 * (x.double().abs() @ w.double().abs().t()) + 64 * U) * (p + one) + half(dt) * gm.abs()
        top = gm.abs() + eg
        within(got[0], gm @ w.double(), eg @ w.double().abs() + (v + 4) * U * (top @ w.double().abs()), dt)
        within(got[1], gm.t() @ x.double(), eg.t() @ x.double().abs() + (rows + 4) * U * (top.t() @ x.double().abs()), dt)
        within(got[2], gm.sum(0), eg.sum(0) + (rows + 4) * U * top.sum(0), dt)
    assert (loss.double() - math.log(v)).abs().max() <= 16 * U * (1 + math.log(v))


def test_cross_entropy_shapes_and_refusals():
    from nirrt_star_amd import nnops
    g = gen(4)
    x, w = randn((2, 5, 8), g, torch.float32), randn((6, 8), g, torch.float32)
    t = torch.randint(0, 6, (2, 5), generator=g, device="cuda")
    per = nnops.linear_cross_entropy(x, w, t, reduction="none")
    assert per.shape == (2, 5)
    want = torch.nn.functional.cross_entropy((x.double() @ w.double().t()).reshape(10, 6), t.reshape(10), reduction="none").view(2, 5)
    assert (per.double() - want).abs().max() < 1e-5
    cw = torch.ones(6, device="cuda")
    for call in (lambda: nnops.linear_cross_entropy(x, w, t.int()), lambda: nnops.linear_cross_entropy(x, w, t[0]),
                 lambda: nnops.linear_cross_entropy(x, w[:, :7], t), lambda: nnops.linear_cross_entropy(x, w[:0], t),
                 lambda: nnops.linear_cross_entropy(x, w, t, bias=cw[:5]), lambda: nnops.linear_cross_entropy(x, w, t, class_weight=cw.double()),
                 lambda: nnops.linear_cross_entropy(x, w, t, class_weight=cw.clone().requires_grad_(True)),
                 lambda: nnops.linear_cross_entropy(x, w, t.cpu()), lambda: nnops.linear_cross_entropy(x, w.half(), t)):
        with pytest.raises(ValueError):
            call()


def test_cross_entropy_in_pieces_of_the_classes():
    """enough rows and classes that the gradient is made piece by piece (its values at a time are bounded): dx sums over the pieces"""
    from nirrt_star_amd import nnops
    g = gen(8)
    rows, k, v = 16000, 8, 9001
    x, w = randn((rows, k), g, torch.bfloat16), randn((v, k), g, torch.bfloat16)
    t = torch.randint(0, v, (rows,), generator=g, device="cuda")
    leaves = [q.clone().requires_grad_(True) for q in (x, w)]
    loss = nnops.linear_cross_entropy(leaves[0], leaves[1], t, reduction="sum")
    got = torch.autograd.grad(loss, leaves)
    dx, dw, total = torch.empty(rows, k, dtype=torch.float64, device="cuda"), torch.zeros(v, k, dtype=torch.float64, device="cuda"), 0.0
    for part in torch.arange(rows, device="cuda").split(2000):
        l = x[part].double() @ w.double().t()
        lp = torch.log_softmax(l, 1)
        total -= float(lp.gather(1, t[part][:, None]).sum())
        p = lp.exp()
        p[torch.arange(len(part)), t[part]] -= 1
        dx[part] = p @ w.double()
        dw += p.t() @ x[part].double()
    assert abs(float(loss) - total) <= 1e-5 * total
    # g is rounded to bf16 (2^-9 of an element), then the result
    h = half(torch.bfloat16)
    assert ((got[0].double() - dx).abs() <= h * (dx.abs() + 3 * w.double().abs().max() * 2) + 1e-4).all()
    assert ((got[1].double() - dw).abs() <= h * dw.abs() + 2 * h * x.double().abs().sum(0).max() / 50 + 1e-3).all()


# ---- norm and clipping -----------------------------------------------------------------------------------------------------------------
def tensor_set(g):
    out = []
    for i, n in enumerate([1, 2, 7, 128, 1000, 4097, 16384, 16385, 50001] * 20):
        out.append(randn((n,), g, TYPES[i % 3], 0.1 * (1 + i % 5)))
    return out


@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e6, float("inf")])
def test_norm_and_clip(max_norm):
    from nirrt_star_amd import nnops
    ts = tensor_set(gen(1)) + [torch.zeros(0, device="cuda")]
    want = math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))
    assert abs(float(nnops.grad_norm(ts)) - want) <= 2 * U * want
    f = min(1.0, max_norm / (want + 1e-6))
    outs = [torch.full(t.shape, 7.0, dtype=TYPES[(i // 3) % 3], device="cuda") for i, t in enumerate(ts)]
    keep = [t.clone() for t in ts]
    norm = nnops.clip_grad_norm_(ts, max_norm, out=outs)
    assert norm.shape == () and abs(float(norm) - want) <= 2 * U * want
    for t, k, o in zip(ts, keep, outs):
        assert torch.equal(t, k)
        within(o, t.double() * f, 6 * U * t.double().abs() * f, o.dtype)
    nnops.clip_grad_norm_(ts, max_norm)
    for t, k in zip(ts, keep):
        within(t, k.double() * f, 6 * U * k.double().abs() * f, t.dtype)
        assert f < 1 or torch.equal(t, k)


def test_norm_special_values_and_layouts():
    from nirrt_star_amd import nnops
    a = torch.randn(300, 40, device="cuda")
    assert float(nnops.grad_norm([torch.zeros(5, device="cuda")])) == 0.0 and float(nnops.grad_norm([torch.zeros(0, device="cuda")])) == 0.0
    z = torch.zeros(5, device="cuda")
    nnops.clip_grad_norm_([z], 1.0)
    assert (z == 0).all()
    big = torch.full((1000,), 1e30, device="cuda")                    # squares beyond fp32
    n = nnops.clip_grad_norm_([big], 1.0)
    assert abs(float(n) / (1e30 * math.sqrt(1000)) - 1) < 1e-6 and abs(float(big.double().norm()) - 1) < 1e-5
    for bad in (float("nan"), float("inf")):
        c = torch.ones(100, device="cuda")
        c[50] = bad
        d = torch.ones(3, device="cuda")
        n = nnops.clip_grad_norm_([c, None, d], 1.0)
        assert not torch.isfinite(n) and (torch.isnan(d).all() if bad != bad else (d == 0).all())
    # not contiguous: the tensor itself is scaled
    base = a.clone()
    view = base.t()[3:17]
    want = view.double().norm()
    assert abs(float(nnops.clip_grad_norm_([view], 1.0)) - float(want)) <= 2 * U * float(want)
    within(base.t()[3:17], a.t()[3:17].double() / (want + 1e-6), 6 * U * (a.t()[3:17].double() / want).abs(), torch.float32)
    assert torch.equal(base[:, :3], a[:, :3]) and torch.equal(base[:, 17:], a[:, 17:])
    # odd addresses
    h = torch.randn(5003, device="cuda").half()
    parts = [h[1:1000], h[1001:1002], h[1003:]]
    want = math.sqrt(sum(float((p.double() ** 2).sum()) for p in parts))
    assert abs(float(nnops.grad_norm(parts)) - want) <= 2 * U * want
    flat = torch.full((5003,), 9.0, device="cuda")
    outs = [flat[1:1000], flat[1001:1002], flat[1003:]]
    nnops.clip_grad_norm_(parts, 1.0, out=outs)
    for p, o in zip(parts, outs):
        within(o, p.double() / (want + 1e-6), 6 * U * p.double().abs() / want, torch.float32)
    assert (flat[[0, 1000, 1002]] == 9).all()


def test_clip_refusals():
    from nirrt_star_amd import nnops
    a, b = torch.ones(8, device="cuda"), torch.ones(8, device="cuda")
    h = torch.ones(8, device="cuda").half()
    for call in (lambda: nnops.clip_grad_norm_([a, a], 1.0), lambda: nnops.clip_grad_norm_([a, b], 1.0, out=[b, a]),
                 lambda: nnops.clip_grad_norm_([a], 1.0, out=[a, b]), lambda: nnops.clip_grad_norm_([a], 1.0, out=[b[:4]]),
                 lambda: nnops.clip_grad_norm_([a], 1.0, out=[torch.ones(8, 2, device="cuda")[:, 0]]),
                 lambda: nnops.clip_grad_norm_([h], 1.0, out=[h.view(torch.bfloat16)]),
                 lambda: nnops.clip_grad_norm_([a, b], 1.0, out=[torch.empty_like(a)] * 2),
                 lambda: nnops.clip_grad_norm_([a, b.double()], 1.0), lambda: nnops.grad_norm([a.to_sparse()]), lambda: nnops.grad_norm([a, b.cpu()])):
        with pytest.raises(ValueError):
            call()
    assert (a == 1).all() and (b == 1).all()
    nnops.clip_grad_norm_([a], 1.0, out=[a])
    assert abs(float(a.norm()) - 1) < 1e-5


# ---- streams and graphs ------------------------------------------------------------------------------------------------------------------
def step(x, w, b, hw, hb, t, cw, flat):
    from nirrt_star_amd import nnops
    h = nnops.linear_act(x, w, b, activation="silu")
    loss = nnops.linear_cross_entropy(h, hw, t, bias=hb, class_weight=cw)
    grads = torch.autograd.grad(loss, [w, b, hw, hb])
    norm = nnops.clip_grad_norm_(grads, 0.05, out=flat)
    return loss, norm


def test_on_another_stream_and_repeatable():
    g = gen(6)
    x, w, b = randn((777, 96), g, torch.float32), randn((130, 96), g, torch.float32, 0.1), randn((130,), g, torch.float32)
    hw, hb = randn((9, 130), g, torch.float32, 0.1), randn((9,), g, torch.float32)
    t, cw = torch.randint(0, 9, (777,), generator=g, device="cuda"), torch.rand(9, generator=g, device="cuda") + 0.5
    for q in (w, b, hw, hb):
        q.requires_grad_(True)
    outs = []
    for i in range(3):
        flat = [torch.empty_like(q) for q in (w, b, hw, hb)]
        st = torch.cuda.Stream() if i else torch.cuda.current_stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            loss, norm = step(x, w, b, hw, hb, t, cw, flat)
        torch.cuda.current_stream().wait_stream(st)
        torch.cuda.synchronize()
        outs.append([loss.detach().clone(), norm.clone()] + [f.clone() for f in flat])
    for o in outs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(outs[0], o))


def test_captured_into_two_graphs_and_replayed():
    g = gen(7)
    data = []
    for rows in (640, 333):
        x, w, b = randn((rows, 64), g, torch.bfloat16), randn((96, 64), g, torch.bfloat16, 0.1), randn((96,), g, torch.bfloat16)
        hw, hb = randn((300, 96), g, torch.bfloat16, 0.1), randn((300,), g, torch.bfloat16)
        t = torch.randint(0, 300, (rows,), generator=g, device="cuda")
        for q in (w, b, hw, hb):
            q.requires_grad_(True)
        data.append((x, w, b, hw, hb, t, None, [torch.empty_like(q, dtype=torch.float32) for q in (w, b, hw, hb)]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for d in data:
            step(*d)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for d in data:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = step(*d)
        graphs.append((gr, res))
    for rep in range(3):
        for d in data:                                   # new inputs in the captured buffers
            d[0].copy_(randn(tuple(d[0].shape), g, torch.bfloat16))
        for gr, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        got = [[r.detach().clone() for r in res] + [f.clone() for f in d[7]] for (_, res), d in zip(graphs, data)]
        for d, q in zip(data, got):
            flat = [torch.empty_like(f) for f in d[7]]
            want = list(step(*d[:7], flat)) + flat
            torch.cuda.synchronize()
            assert all(torch.equal(a, e) for a, e in zip(q, want))


def test_more_than_two_to_the_31_elements():
    """offsets past 32 bits: only the last rows are looked at"""
    from nirrt_star_amd import nnops
    m, k = 70000, 32768
    x = torch.empty(m, k, dtype=torch.float16, device="cuda")
    x[-3:] = randn((3, k), gen(1), torch.float16)
    x[:-3] = 0
    w = randn((3, k), gen(2), torch.float16, 0.01)
    y = nnops.linear_act(x, w)
    _, _, want, ey = linear64(x[-3:], w, None, None, "none")
    within(y[-3:], want, ey, torch.float16)
    assert (y[:-3] == 0).all()
    assert abs(float(nnops.grad_norm([x])) / float(x[-3:].double().norm()) - 1) < 1e-6


# ---- sizes at which the kernels change ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,k,n", [(16, 515, 321), (17, 4096, 40), (32, 7, 16), (33, 515, 321), (31, 1, 4100)])
def test_linear_few_rows(m, k, n, dt):
    test_linear_gradients(m, k, n, "gelu", dt)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,k,n,act", [(4000, 328, 4064, "silu"), (4000, 4064, 328, "gelu"), (328, 4064, 4000, "relu"), (4000, 329, 4063, "silu"),
                                       (4003, 4063, 327, "none"), (3000, 1000, 24, "none"), (300, 9000, 264, "gelu"), (777, 515, 1029, "none")])
def test_linear_large_tiles_and_parts(m, k, n, act, dt):
    """the largest tiles in each of the three products with ragged edges, reductions in parts, odd operands copied into whole chunks"""
    if act == "relu":                  # (no slope at a rounded 0: the forward product only)
        from nirrt_star_amd import nnops
        g = gen(m + k)
        x, w, b = randn((m, k), g, dt), randn((n, k), g, dt, k ** -0.5), randn((n,), g, dt)
        _, _, y, ey = linear64(x, w, b, None, act)
        within(nnops.linear_act(x, w, b, activation=act), y, ey, dt)
        act = "silu"
    test_linear_gradients(m, k, n, act, dt)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ["none", "silu"])
def test_linear_layouts_of_the_incoming_gradient(act, dt):
    """gradients that arrive transposed, as columns of a wider tensor, off 16 bytes, or as one value for all (a sum's)"""
    g = gen(17)
    for m, k, n in ((70, 40, 48), (129, 33, 35)):
        for dy in (randn((n, m), g, dt).t(), randn((m, n + 9), g, dt)[:, 3:3 + n], randn((m, 2 * n), g, dt)[:, ::2], randn((1, 1), g, dt).expand(m, n),
                   randn((1, n), g, dt).expand(m, n)):
            test_linear_gradients(m, k, n, act, dt, dy)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,k,v", [(64, 31, 3), (256, 128, 5), (257, 200, 8), (255, 129, 9), (128, 64, 64), (130, 8, 65), (2100, 515, 1031), (3000, 264, 4100),
                                      (33, 1030, 257), (1500, 1, 6)])
def test_cross_entropy_more_sizes(rows, k, v, dt):
    test_cross_entropy(rows, k, v, "mean", True, True, dt)
    test_cross_entropy(rows, k, v, "none", False, False, dt)
