"""GPU: calls of nirrt_star_amd.nnops that its documentation allows beyond sizes and types (test_nnops_gpu.py has those): operands far apart,
losses and gradients used in place, autocast, the largest dimensions."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, g, dt, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt)


# ---- cross entropy: operands of any stride -----------------------------------------------------------------------------------------------
def spread(t, row_bytes, shift=0):
    """t's values in rows that lie row_bytes apart, from element `shift` on"""
    ld = row_bytes // t.element_size()
    flat = torch.zeros(t.shape[0] * ld + shift, dtype=t.dtype, device=t.device)
    v = flat[shift:].as_strided(t.shape, (ld, 1), shift)
    v.copy_(t)
    return v


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("classes", [7, 33])
@pytest.mark.parametrize("k", [64, 61])
def test_cross_entropy_operands_of_any_stride(dt, classes, k):
    """rows apart by less and more than the 4 MB that the products read directly, off 16 bytes, padded, transposed: what the kernels multiply is
    the same in all of them, so the bits are those of contiguous operands"""
    from nirrt_star_amd import nnops
    g = gen(k + classes)
    rows = 9
    x, w, b = randn((rows, k), g, dt), randn((classes, k), g, dt), randn((classes,), g, dt)
    t = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    t[4] = -100

    def run(x, w):
        leaves = [x.detach().requires_grad_(True), w.detach().requires_grad_(True)]
        loss = nnops.linear_cross_entropy(leaves[0], leaves[1], t, bias=b)
        return [loss.detach()] + list(torch.autograd.grad(loss, leaves))

    want = run(x, w)
    assert all(torch.isfinite(q).all() for q in want)
    xs = [spread(x, 1 << 12), spread(x, 1 << 22), spread(x, (1 << 22) + 16), spread(x, 1 << 24, 3), spread(x, 1 << 10, 1), x.t().contiguous().t()]
    ws = [spread(w, 1 << 22), spread(w, (1 << 22) + 16), spread(w, 1 << 23, 1), spread(w, 1 << 10, 1), w.t().contiguous().t()]
    for q in xs:
        assert all(torch.equal(a, e) for a, e in zip(run(q, w), want))
    for q in ws:
        assert all(torch.equal(a, e) for a, e in zip(run(x, q), want))
    assert all(torch.equal(a, e) for a, e in zip(run(xs[3], ws[2]), want))


def test_cross_entropy_of_the_last_token():
    from nirrt_star_amd import nnops
    g = gen(2)
    h = torch.zeros(5, 1030, 2048, dtype=torch.bfloat16, device="cuda")
    h[:, -1] = randn((5, 2048), g, torch.bfloat16)
    w, t = randn((100, 2048), g, torch.bfloat16, 0.02), torch.arange(5, device="cuda") * 7
    h.requires_grad_(True)
    loss = nnops.linear_cross_entropy(h[:, -1], w, t, reduction="sum")
    dh, = torch.autograd.grad(loss, h)
    last = h[:, -1].detach().contiguous().requires_grad_(True)
    want = nnops.linear_cross_entropy(last, w, t, reduction="sum")
    d, = torch.autograd.grad(want, last)
    assert torch.equal(loss, want) and torch.equal(dh[:, -1], d) and (dh[:, :-1] == 0).all()


# ---- forward mode and traces ---------------------------------------------------------------------------------------------------------------
def test_dual_numbers_are_refused_where_a_tangent_would_be_lost():
    from torch.autograd import forward_ad
    from nirrt_star_amd import nnops
    x, w, t = torch.randn(5, 4, device="cuda"), torch.randn(3, 4, device="cuda"), torch.zeros(5, dtype=torch.int64, device="cuda")
    plain = nnops.linear_act(x, w, activation="silu")
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: nnops.linear_act(d, w), lambda: nnops.linear_act(x, forward_ad.make_dual(w, torch.ones_like(w))),
                     lambda: nnops.linear_act(x, w, residual=forward_ad.make_dual(plain, torch.ones_like(plain))),
                     lambda: nnops.linear_cross_entropy(d, w, t), lambda: nnops.grad_norm([x, d]), lambda: nnops.clip_grad_norm_([d], 1.0)):
            with pytest.raises(NotImplementedError):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
        assert torch.equal(nnops.linear_act(x, w, activation="silu"), plain)         # (no dual number: as everywhere)
    assert (d == x).all()


def test_traces_are_refused():
    from nirrt_star_amd import nnops
    x, w = torch.randn(5, 4, device="cuda"), torch.randn(3, 4, device="cuda", requires_grad=True)
    for weight in (w, w.detach()):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(lambda q: nnops.linear_act(q, weight), (x,), check_trace=False)


# ---- in place on results and on saved tensors ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("classes", [2, 40])
def test_the_loss_can_be_changed_in_place(reduction, classes):
    """loss /= steps; loss += another term: as on any loss"""
    from nirrt_star_amd import nnops
    g = gen(classes)
    x, w = randn((30, 16), g, torch.float32), randn((classes, 16), g, torch.float32)
    t = torch.randint(0, classes, (30,), generator=g, device="cuda")
    cw = torch.rand(classes, generator=g, device="cuda") + 0.5

    def leaves():
        return [q.clone().requires_grad_(True) for q in (x, w)]

    a, b = leaves(), leaves()
    want = nnops.linear_cross_entropy(a[0], a[1], t, class_weight=cw, reduction=reduction)
    value = want.detach().clone()
    (want / 4 + (a[0] ** 2).sum()).sum().backward()
    loss = nnops.linear_cross_entropy(b[0], b[1], t, class_weight=cw, reduction=reduction)
    loss /= 4
    loss += (b[0] ** 2).sum()
    loss.sum().backward()
    assert torch.equal(loss.detach(), value / 4 + (x ** 2).sum())
    for p, q in zip(a, b):
        assert torch.equal(p.grad, q.grad)
    total = torch.zeros((), device="cuda")
    total += nnops.linear_cross_entropy(x, w, t, class_weight=cw, reduction="sum")
    assert float(total) > 0


def test_clipping_is_seen_by_graphs_that_saved_the_tensor():
    from nirrt_star_amd import nnops
    x = torch.ones(8, device="cuda", requires_grad=True)
    wide = torch.ones(8, 3, device="cuda")
    for g, out in ((torch.full((8,), 3.0, device="cuda"), None), (wide[:, 1], None), (torch.ones(8, device="cuda"), torch.zeros(8, device="cuda"))):
        saved = g if out is None else out
        y = (x * saved).sum()                       # keeps `saved` for x's gradient
        before = saved._version
        nnops.clip_grad_norm_([None, g], 0.5, out=None if out is None else [None, out])
        assert saved._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():                    # (tensors without a version)
        g = torch.full((8,), 3.0, device="cuda")
        nnops.clip_grad_norm_([g], 1.0)
        assert abs(float(g.norm()) - 1) < 1e-5


def test_clipping_refuses_parameters():
    from nirrt_star_amd import nnops
    model = torch.nn.Linear(6, 4).cuda()
    model(torch.randn(3, 6, device="cuda")).sum().backward()
    before = [p.detach().clone() for p in model.parameters()]
    grads = [p.grad for p in model.parameters()]
    with pytest.raises(ValueError, match="not the parameters"):
        nnops.clip_grad_norm_(model.parameters(), 1.0)
    with pytest.raises(ValueError, match="not the parameters"):
        nnops.clip_grad_norm_(grads, 1.0, out=list(model.parameters()))
    assert all(torch.equal(p, q) for p, q in zip(model.parameters(), before))
    assert float(nnops.grad_norm(model.parameters())) > 0                 # (reading them is fine)
    nnops.clip_grad_norm_(grads, 1.0)
    assert abs(float(nnops.grad_norm(grads)) - 1) < 1e-5
    # gradients that carry a graph of their own are no leaves
    x = torch.randn(5, device="cuda", requires_grad=True)
    g, = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    assert g.requires_grad
    nnops.clip_grad_norm_([g], 1.0)
    assert abs(float(nnops.grad_norm([g])) - 1) < 1e-5


# ---- special values --------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("with_res", [False, True])
def test_a_nan_before_the_activation_reaches_the_gradients(act, dt, with_res):
    """row 2 of x is NaN: its pre-activations, values and slopes are; the other rows' dx do not see it, dw and db (sums over the rows) do"""
    from nirrt_star_amd import nnops
    g = gen(5)
    x, w, b, r = randn((40, 16), g, dt), randn((24, 16), g, dt), randn((24,), g, dt), randn((40, 24), g, dt)
    x[2, 3] = float("nan")
    leaves = [q.clone().requires_grad_(True) for q in (x, w, b)]
    y = nnops.linear_act(*leaves, residual=r if with_res else None, activation=act)
    dx, dw, db = torch.autograd.grad(y, leaves, torch.ones_like(y))
    rest = torch.arange(40, device="cuda") != 2
    assert torch.isnan(y[2]).all() and torch.isfinite(y[rest]).all()
    assert torch.isnan(dx[2]).all() and torch.isfinite(dx[rest]).all() and torch.isnan(dw).all() and torch.isnan(db).all()


# ---- the largest dimensions --------------------------------------------------------------------------------------------------------------------
MOST = (1 << 31) - 4096


def test_the_longest_reduction():
    """few rows: whole numbers, so the sum is exact whatever its order"""
    from nirrt_star_amd import nnops
    x, w = (torch.zeros(1, MOST, dtype=torch.float16, device="cuda") for _ in range(2))
    at = torch.tensor([0, 1, 2047, 2048, 1 << 30, MOST - 2049, MOST - 2048, MOST - 257, MOST - 256, MOST - 1], device="cuda")
    x[0, at] = torch.arange(1, 11, device="cuda").half()
    w[0, at] = 2.0
    assert float(nnops.linear_act(x, w)) == 110.0
    with pytest.raises(ValueError, match="beyond"):
        nnops.linear_act(torch.empty(0, MOST + 1, device="cuda"), torch.empty(0, MOST + 1, device="cuda"))


def test_column_sums_of_the_most_rows():
    from nirrt_star_amd import nnops
    L = nnops._lib()
    dy = torch.zeros(MOST, 8, dtype=torch.float16, device="cuda")
    at = torch.tensor([0, 255, 256, 1023, 1024, 1 << 30, MOST - 1025, MOST - 1024, MOST - 256, MOST - 1], device="cuda")
    dy[at] = (torch.arange(80, device="cuda") % 13).view(10, 8).half()
    db = torch.empty(8, dtype=torch.float16, device="cuda")
    ws = torch.empty(L.nirrt_nn_linear_backward_workspace(2, 0, None, 8, None, 8, dy.data_ptr(), 8, MOST, 8, 0), dtype=torch.uint8, device="cuda")
    assert L.nirrt_nn_linear_backward(2, 0, None, 8, None, 8, None, dy.data_ptr(), 8, None, None, db.data_ptr(), MOST, 8, 0, ws.data_ptr(),
                                      torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(db, (torch.arange(80, device="cuda") % 13).view(10, 8).sum(0).half())


def test_more_rows_and_columns_than_a_launch_has_small_tiles_for():
    """2^30 + 5 rows of a narrow layer, 2^27 + 5 columns for two rows: whole numbers, looked at in a few places"""
    from nirrt_star_amd import nnops
    g = gen(6)
    for m, n, k in (((1 << 30) + 5, 3, 8), (2, (1 << 27) + 5, 8)):
        x, w = torch.zeros(m, k, dtype=torch.float16, device="cuda"), torch.zeros(n, k, dtype=torch.float16, device="cuda")
        at, long = torch.tensor([0, 1, 63, 64, 1 << 26, max(m, n) - 6, max(m, n) - 5, max(m, n) - 1], device="cuda"), x if m > n else w
        short = w if m > n else x
        long[at] = torch.randint(-3, 4, (8, k), generator=g, device="cuda").half()
        short.copy_(torch.randint(-3, 4, tuple(short.shape), generator=g, device="cuda"))
        y = nnops.linear_act(x, w)
        got = y[at] if m > n else y[:, at].t()
        assert torch.equal(got.double(), long[at].double() @ short.double().t())
        assert int((y != 0).sum()) == int((got != 0).sum())
        del x, w, long, short, y


# ---- workspaces ----------------------------------------------------------------------------------------------------------------------------------
def test_cross_entropy_holds_no_copies_that_are_not_made():
    from nirrt_star_amd import nnops
    g = gen(3)
    rows, k, classes = 64, 512, 50000
    x, w = randn((rows, k), g, torch.bfloat16).requires_grad_(True), randn((classes, k), g, torch.bfloat16, 0.05)
    t = torch.randint(0, classes, (rows,), generator=g, device="cuda")

    def more(call):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        out = call()
        torch.cuda.synchronize()
        return torch.cuda.max_memory_allocated() - held, out

    for weight in (w, w.detach()[:, :500]):                         # (51 MB each; rows of 1000 bytes are copied)
        xx = x[:, :weight.shape[1]]
        extra, loss = more(lambda: nnops.linear_cross_entropy(xx, weight, t))
        assert extra < (4 << 20) + (0 if weight is w else 51 << 20)
        extra, _ = more(lambda: torch.autograd.grad(loss, x))       # g' is rows x classes
        assert extra < (4 << 20) + rows * classes * 2 + 32 * rows * k * 4 + (0 if weight is w else 51 << 20)
    x2 = randn((1 << 20, 128), g, torch.float32)                    # two classes: sums of the workgroups only
    extra, _ = more(lambda: nnops.linear_cross_entropy(x2, randn((2, 128), g, torch.float32), torch.zeros(1 << 20, dtype=torch.int64, device="cuda")))
    assert extra < (8 << 20) + (1 << 20) * (8 + 4 + 8)


@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("far_x", [False, True])
@pytest.mark.parametrize("far_w", [False, True])
def test_cross_entropy_workspaces_without_the_copies(dt, far_x, far_w):
    """the C entry points with exactly the bytes they need, and marked bytes behind them that have to stay"""
    from nirrt_star_amd import nnops
    L = nnops._lib()
    g = gen(dt)
    T = TYPES[dt]
    rows, k, classes = 300, 64, 700
    x, w = randn((rows, k), g, T), randn((classes, k), g, T)
    if far_x:
        x = spread(x, 1 << 10, 1)
    if far_w:
        w = spread(w, 1 << 10, 1)
    t = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    X, W = (r * k * T.itemsize + 255 & ~255 for r in (rows, classes))
    st = torch.cuda.current_stream().cuda_stream

    def space(nbytes):
        return torch.full((nbytes + 4096,), 0x5a, dtype=torch.uint8, device="cuda")

    def outs():
        return (torch.empty(rows, 2, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(3, device="cuda"), torch.empty(rows, k, dtype=T, device="cuda"),
                torch.empty(classes, k, dtype=T, device="cuda"), torch.empty(classes, dtype=T, device="cuda"))

    one = torch.ones((), device="cuda")
    res = []
    for short in (False, True):
        lse, nll, total, dx, dw, db = o = outs()
        n = L.nirrt_nn_cross_entropy_workspace(dt, rows, classes, k) - ((0 if far_x else X) + (0 if far_w else W) if short else 0)
        ws = space(n)
        assert L.nirrt_nn_cross_entropy(dt, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), None, t.data_ptr(), None, -100, lse.data_ptr(), nll.data_ptr(),
                                        total.data_ptr(), rows, classes, k, ws.data_ptr(), st) == 0
        assert (ws[n:] == 0x5a).all()
        n = L.nirrt_nn_cross_entropy_backward_workspace(dt, rows, classes, k) - ((0 if far_w else W) if short else 0)
        ws = space(n)
        assert L.nirrt_nn_cross_entropy_backward(dt, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), None, t.data_ptr(), None, -100, lse.data_ptr(),
                                                 one.data_ptr(), 0, total.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), rows, classes, k, ws.data_ptr(), st) == 0
        assert (ws[n:] == 0x5a).all()
        res.append(o)
    assert all(torch.equal(p, q) and torch.isfinite(p).all() for p, q in zip(*res))


def test_c_backward_of_a_layer_without_outputs():
    """n = 0 through the C entry: dx is zero, dw and db are empty"""
    from nirrt_star_amd import nnops
    L = nnops._lib()
    x, dx = torch.randn(40, 16, device="cuda"), torch.full((40, 16), 7.0, device="cuda")
    for act in range(4):
        need = L.nirrt_nn_linear_backward_workspace(0, act, x.data_ptr(), 16, None, 16, None, 0, 40, 0, 16)
        ws = torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")
        for db in (None, ws.data_ptr()):
            dx.fill_(7.0)
            assert L.nirrt_nn_linear_backward(0, act, x.data_ptr(), 16, None, 16, None, None, 0, dx.data_ptr(), ws.data_ptr(), db, 40, 0, 16, ws.data_ptr(),
                                              torch.cuda.current_stream().cuda_stream) == 0
            assert (dx == 0).all()


@pytest.mark.parametrize("classes", [5, 30])
def test_cross_entropy_without_inputs_has_a_bias_gradient(classes):
    from nirrt_star_amd import nnops
    g = gen(classes)
    b = randn((classes,), g, torch.float32).requires_grad_(True)
    x, w = torch.zeros(20, 0, device="cuda", requires_grad=True), torch.zeros(classes, 0, device="cuda", requires_grad=True)
    t = torch.randint(0, classes, (20,), generator=g, device="cuda")
    dx, dw, db = torch.autograd.grad(nnops.linear_cross_entropy(x, w, t, bias=b, reduction="sum"), (x, w, b))
    want = 20 * torch.softmax(b.detach().double(), 0) - torch.bincount(t, minlength=classes)
    # 20 terms below 1, each off by a few 2^-24 (exp, lse), and their sum
    assert dx.shape == x.shape and dw.shape == w.shape and (db.double() - want).abs().max() <= 20 * 64 * 2.0 ** -24
