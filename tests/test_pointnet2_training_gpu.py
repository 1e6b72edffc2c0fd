"""GPU: a training step of the guidance network (pointnet2.train_step): head + loss, gradients' norm and clipping used together, against the
plain evaluation of the same step."""
import copy

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _batch(B, N, seed):
    rng = np.random.RandomState(seed)
    xyz = rng.uniform(-0.7, 0.7, (B, 3, N))
    xyz[:, 2] = 0
    start = (np.abs(xyz[:, 0] + 0.5) < 0.1).astype(np.float64)
    goal = (np.abs(xyz[:, 0] - 0.5) < 0.1).astype(np.float64)
    x = np.concatenate([xyz, start[:, None], goal[:, None], ((start + goal) == 0)[:, None]], axis=1).astype(np.float32)
    labels = (np.abs(xyz[:, 1]) < 0.15).astype(np.int64)
    labels[:, :5] = -100
    starts = [torch.from_numpy(rng.randint(0, m, B)) for m in (N, 1024, 256, 64)]
    return torch.from_numpy(x).cuda(), torch.from_numpy(labels).cuda(), starts


def _model(seed=0):
    from nirrt_star_amd.pointnet2 import get_model
    torch.manual_seed(seed)
    m = get_model(2).cuda().train()
    m.drop1.p = 0.0                 # (the plain evaluation below has to see the same features)
    return m


def test_step_equals_the_plain_evaluation():
    from nirrt_star_amd.pointnet2 import train_step
    m = _model()
    x, labels, starts = _batch(2, 1500, 1)
    cw = torch.tensor([1.0, 1.7], device="cuda")
    seen = {}
    hook = m.bn1.register_forward_hook(lambda mod, i, o: seen.__setitem__("h", o.detach()))
    before = {k: p.detach().clone() for k, p in m.named_parameters()}
    opt = torch.optim.SGD(m.parameters(), lr=1.0)
    loss, norm = train_step(m, opt, x, labels, cw, max_norm=0.25, fps_starts=starts)
    hook.remove()
    # head and loss from the features the step saw, in 64 bits
    h = seen["h"].relu().double()
    w, b = before["conv2.weight"].squeeze(2).double(), before["conv2.bias"].double()
    t = labels.reshape(-1)
    keep = t >= 0
    logp = torch.log_softmax(h @ w.t() + b, 1)
    wt = cw.double()[t[keep]]
    want = -(logp[keep, t[keep]] * wt).sum() / wt.sum()
    assert abs(float(loss) - float(want)) <= 130 * 2.0 ** -24 * (1 + float((h.abs() @ w.abs().t()).max()))
    g = logp.exp()
    g[keep, t[keep]] -= 1
    g = torch.where(keep[:, None], g * (cw.double()[t.clamp(min=0)] / wt.sum())[:, None], torch.zeros_like(g))
    grads = {k: p.grad for k, p in m.named_parameters()}
    assert all(v is not None and torch.isfinite(v).all() for v in grads.values()) and len(grads) == 138
    # .grad holds the clipped gradients; the norm was taken before
    f = min(1.0, 0.25 / (float(norm) + 1e-6))
    total = float(torch.stack([v.double().square().sum() for v in grads.values()]).sum().sqrt())
    assert f < 1 and abs(total - 0.25) <= 1e-5
    bound = (len(t) + 140) * 2.0 ** -24
    dw, db = (g.t() @ h) * f, g.sum(0) * f
    assert ((grads["conv2.weight"].squeeze(2).double() - dw).abs() <= bound * f * (g.abs().t() @ h.abs()) + 1e-6 * dw.abs()).all()
    assert ((grads["conv2.bias"].double() - db).abs() <= bound * f * g.abs().sum(0) + 1e-6 * db.abs()).all()
    # the optimiser stepped with them
    for k, p in m.named_parameters():
        assert torch.equal(p.detach(), before[k] - grads[k])


def test_gradients_of_all_layers_agree_with_the_reference_loss():
    """the same loss through log_softmax and F.nll_loss: gradients of every layer, compared in the 2-norm (gathers add with atomics in
    torch's backward pass, so the last bits differ from run to run; BatchNorm's division by small deviations spreads them: 1e-3)"""
    m = _model(3)
    ref = copy.deepcopy(m)
    x, labels, starts = _batch(3, 1200, 2)
    cw = torch.tensor([1.0, 2.5], device="cuda")
    m.loss(x, labels, cw, starts).backward()
    logp, _ = ref(x, fps_starts=starts)
    torch.nn.functional.nll_loss(logp.reshape(-1, 2), labels.reshape(-1), weight=cw).backward()
    num = den = 0.0
    for (k, p), (_, q) in zip(m.named_parameters(), ref.named_parameters()):
        num += float((p.grad.double() - q.grad.double()).square().sum())
        den += float(q.grad.double().square().sum())
    assert num <= 1e-6 * den


def test_without_clipping_the_gradients_stay():
    from nirrt_star_amd.pointnet2 import train_step
    m = _model(5)
    x, labels, starts = _batch(1, 1100, 4)
    opt = torch.optim.SGD(m.parameters(), lr=0.0)
    loss, norm = train_step(m, opt, x, labels, fps_starts=starts)
    total = float(torch.stack([p.grad.double().square().sum() for p in m.parameters()]).sum().sqrt())
    assert torch.isfinite(loss) and abs(float(norm) - total) <= 1e-6 * total


def test_a_folded_model_in_eval_mode_is_refused():
    m = _model(6).eval().fold()
    x, labels, starts = _batch(1, 1100, 4)
    with pytest.raises(RuntimeError):
        m.loss(x, labels)
    m.train()
    assert torch.isfinite(m.loss(x, labels, None, starts))


def test_a_capture_is_refused_before_anything_is_recorded():
    from nirrt_star_amd.pointnet2 import train_step
    m = _model(7)
    x, labels, starts = _batch(1, 1100, 4)
    opt = torch.optim.SGD(m.parameters(), lr=1.0)
    y, side = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError):
            train_step(m, opt, x, labels, fps_starts=starts)
        y.copy_(side + 1)
    assert all(p.grad is None for p in m.parameters())
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert (y == 1).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_loss_under_autocast(dt):
    """the layers before the head in 16 bits, the head and the loss as without autocast; gradients in the parameters' type"""
    m = _model(8)
    x, labels, starts = _batch(2, 1300, 5)
    cw = torch.tensor([1.0, 1.7], device="cuda")
    seen = {}
    hook = m.bn1.register_forward_hook(lambda mod, i, o: seen.__setitem__("h", o.detach()))
    with torch.autocast("cuda", dtype=dt):
        loss = m.loss(x, labels, cw, starts)
        hook.remove()
        assert m(x, fps_starts=starts)[0].shape == (2, 1300, 2)            # (what the loss replaces works there too)
    loss.backward()
    h = seen["h"].relu().double()
    w, b = m.conv2.weight.squeeze(2).detach().double(), m.conv2.bias.detach().double()
    t = labels.reshape(-1)
    keep = t >= 0
    logp = torch.log_softmax(h @ w.t() + b, 1)
    wt = cw.double()[t[keep]]
    want = -(logp[keep, t[keep]] * wt).sum() / wt.sum()
    assert loss.dtype == torch.float32 and seen["h"].dtype == torch.float32
    assert abs(float(loss.detach()) - float(want)) <= 130 * 2.0 ** -24 * (1 + float((h.abs() @ w.abs().t()).max()))
    assert all(p.grad is not None and p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all() for p in m.parameters())
