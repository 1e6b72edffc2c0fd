"""The dense operators of the guidance network's layers and of a training step, as cases to time and compare.

Three operators (nirrt_star_amd.nnops): `linear_act` = act(x W^T + b) + r with its backward pass, `linear_cross_entropy` = a classification head
with softmax cross entropy and its gradient, `clip_grad_norm_` = the global norm over many tensors and clipping.  `own = False`
computes them in elementary torch operations in 32 bits, `own = True` through the package."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def _linear(name, rows, k, n, dtype, act, residual, train):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "act": act, "residual": residual, "train": train}


def _ce(name, rows, k, classes, dtype, bias, weighted):
    return {"name": name, "op": "ce", "rows": rows, "k": k, "classes": classes, "dtype": dtype, "bias": bias, "weighted": weighted}


def _clip(name, tensors, elements, dtype, out_dtype):
    return {"name": name, "op": "clip", "tensors": tensors, "elements": elements, "dtype": dtype, "out_dtype": out_dtype}


def listed():
    return [
        # one point through a 128-wide layer: only latency counts
        _linear("one_row", 1, 128, 128, "fp32", "relu", False, False),
        # the last feature-propagation layer of the guidance network over one cloud of 2048 points
        _linear("cloud_layer", 2048, 128, 128, "fp32", "relu", False, False),
        # the first layer of the fourth set-abstraction level for a refresh of 256 clouds (16 groups of 32 members, 512 + 3 + 1 inputs)
        _linear("refresh_layer", 131072, 516, 256, "fp32", "relu", False, False),
        # a few rows through a wide layer: every weight is read for them
        _linear("few_rows_wide", 7, 4096, 4096, "fp16", "silu", True, False),
        # a training step of a feature-propagation layer (352 -> 256) over 32 clouds
        _linear("train_layer", 32768, 352, 256, "fp32", "gelu", False, True),
        # odd widths, forward and backward
        _linear("train_odd", 4097, 321, 515, "bf16", "gelu", True, True),
        # a wide layer in training: the largest product
        _linear("train_wide", 16384, 4096, 4096, "bf16", "silu", True, True),
        # the guidance network's head and loss in training: path / no path, class weights of the training set
        _ce("two_classes", 32768, 128, 2, "fp32", True, True),
        # odd widths, some rows ignored
        _ce("classes_odd", 513, 771, 5003, "fp16", True, False),
        # a large set of classes: the logits alone would be a gigabyte in 32 bits
        _ce("many_classes", 8192, 1024, 32003, "bf16", False, False),
        # the gradients of the guidance network (1.9 M parameters in 132 tensors)
        _clip("net_gradients", 132, 1880000, "fp32", "fp32"),
        # half-precision gradients of a large model, clipped into 32-bit ones
        _clip("large_gradients", 300, 260000000, "bf16", "fp32"),
    ]


def _log_int(rng, lo, hi):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return max(lo, min(hi, int(v)))


def draw(rng):
    op = rng.choice(["linear", "linear", "ce", "clip"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "linear":
        train = rng.random() < 0.5
        while True:
            rows, k, n = _log_int(rng, 1, 131072), _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)
            # (32-bit products run at a sixteenth of the 16-bit rate: less work than the largest listed case)
            if rows * k * n * (3 if train else 1) <= (4e10 if dtype == "fp32" else 6e11):
                break
        # half of the widths are multiples of eight, as layers mostly have them
        if rng.random() < 0.5:
            k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
        # (a rectified layer's gradient jumps where z changes sign, which the last bit of a sum decides: smooth ones in training)
        act = rng.choice(["none", "gelu", "silu"] if train else ["none", "relu", "gelu", "silu"])
        return {"op": op, "rows": rows, "k": k, "n": n, "dtype": dtype, "act": act, "residual": rng.random() < 0.5, "train": train}
    if op == "ce":
        while True:
            rows, k, classes = _log_int(rng, 16, 65536), _log_int(rng, 16, 2048), _log_int(rng, 2, 65536)
            if rows * k * classes <= (3e10 if dtype == "fp32" else 2.6e11) and rows * classes <= 260000000:
                break
        if rng.random() < 0.5:
            k = (k + 7) // 8 * 8
        return {"op": op, "rows": rows, "k": k, "classes": classes, "dtype": dtype, "bias": rng.random() < 0.5, "weighted": rng.random() < 0.5}
    tensors = _log_int(rng, 1, 600)
    return {"op": op, "tensors": tensors, "elements": max(tensors, _log_int(rng, 1000, 200000000)), "dtype": dtype,
            "out_dtype": rng.choice([dtype, "fp32"])}


def _sizes(case):
    """sizes of the gradient tensors: spread over three decades, odd ones among them, `elements` in all"""
    n, total = case["tensors"], case["elements"]
    weights = [math.exp(7.0 * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]
    sizes = [1 + int(w / sum(weights) * (total - n)) for w in weights]
    sizes[0] += total - sum(sizes)
    return sizes


def _randn(shape, g, dtype, scale=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, scale, generator=g).to(DTYPES[dtype])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "linear":
        m, k, n, dt = case["rows"], case["k"], case["n"], case["dtype"]
        st = {"case": case, "x": _randn((m, k), g, dt), "w": _randn((n, k), g, dt, k ** -0.5), "b": _randn((n,), g, dt, 0.1),
              "r": _randn((m, n), g, dt) if case["residual"] else None}
        if case["train"]:
            st["dy"] = _randn((m, n), g, dt)
            for key in ("x", "w", "b", "r"):
                if st[key] is not None:
                    st[key].requires_grad_(True)
        return st
    if case["op"] == "ce":
        m, k, v, dt = case["rows"], case["k"], case["classes"], case["dtype"]
        st = {"case": case, "x": _randn((m, k), g, dt), "w": _randn((v, k), g, dt, 1.5 * k ** -0.5),
              "b": _randn((v,), g, dt, 0.5) if case["bias"] else None,
              "cw": torch.empty(v, device="cuda").uniform_(1.0, 3.0, generator=g) if case["weighted"] else None}
        t = torch.randint(0, v, (m,), generator=g, device="cuda")
        # a tenth of the rows is ignored (never all of them)
        skip = torch.rand(m, generator=g, device="cuda") < 0.1
        skip[0] = False
        st["t"] = torch.where(skip, torch.full_like(t, -100), t)
        for key in ("x", "w", "b"):
            if st[key] is not None:
                st[key].requires_grad_(True)
        return st
    # gradients as a step leaves them: magnitudes differ from tensor to tensor; the clipped ones go into one flat buffer, as an
    # optimiser that updates all parameters at once keeps it
    sizes = _sizes(case)
    scale = torch.exp(torch.empty(len(sizes)).uniform_(-3.0, 0.0, generator=torch.Generator().manual_seed(seed))).tolist()
    grads = [_randn((s,), g, case["dtype"], 0.05 * f) for s, f in zip(sizes, scale)]
    flat = torch.empty(sum(sizes), dtype=DTYPES[case["out_dtype"]], device="cuda")
    return {"case": case, "grads": grads, "flat": flat, "out": list(flat.split(sizes))}


def _act(z, name):
    if name == "none":
        return z
    if name == "relu":
        return torch.clamp(z, min=0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.7071067811865476))
    return z / (1 + torch.exp(-z))


def _act_grad(z, name):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.7071067811865476)) + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _plain_linear(st, ft, ot):
    c = st["case"]
    x, w, b = st["x"].detach().to(ft), st["w"].detach().to(ft), st["b"].detach().to(ft)
    z = x @ w.t() + b
    y = _act(z, c["act"])
    if st["r"] is not None:
        y = y + st["r"].detach().to(ft)
    if not c["train"]:
        return {"y": y.to(ot)}
    dy = st["dy"].to(ft)
    dz = dy * _act_grad(z, c["act"])
    out = {"y": y.to(ot), "dx": (dz @ w).to(ot), "dw": (dz.t() @ x).to(ot), "db": dz.sum(0).to(ot)}
    if st["r"] is not None:
        out["dr"] = dy.to(ot)
    return out


def _plain_ce(st):
    x, w = st["x"].detach().float(), st["w"].detach().float()
    t, ot = st["t"], st["x"].dtype
    logits = x @ w.t()
    if st["b"] is not None:
        logits = logits + st["b"].detach().float()
    m = logits.max(dim=1, keepdim=True)[0]
    e = torch.exp(logits - m)
    s = e.sum(dim=1, keepdim=True)
    keep = t >= 0
    ts = torch.where(keep, t, torch.zeros_like(t))
    wt = keep.float() if st["cw"] is None else torch.where(keep, st["cw"][ts], torch.zeros_like(st["cw"][ts]))
    nll = (m + torch.log(s)).squeeze(1) - logits.gather(1, ts[:, None]).squeeze(1)
    total = wt.sum()
    loss = (nll * wt).sum() / total
    coef = (wt / total)[:, None]
    gmat = e / s * coef
    gmat.scatter_add_(1, ts[:, None], -coef)
    out = {"loss": loss, "dx": (gmat @ w).to(ot), "dw": (gmat.t() @ x).to(ot)}
    if st["b"] is not None:
        out["db"] = gmat.sum(0).to(ot)
    return out


def _plain_clip(st, max_norm):
    total = torch.stack([g.float().square().sum() for g in st["grads"]]).sum()
    norm = total.sqrt()
    scale = torch.clamp(max_norm / (norm + 1e-6), max=1.0)
    for g, o in zip(st["grads"], st["out"]):
        o.copy_(g.float() * scale)
    return {"norm": norm, "out": st["flat"]}


MAX_NORM = 1.0


def run(state):
    op = state["case"]["op"]
    if not own:
        if op == "linear":
            return _plain_linear(state, torch.float32, state["x"].dtype)
        if op == "ce":
            return _plain_ce(state)
        return _plain_clip(state, MAX_NORM)
    from nirrt_star_amd import nnops
    if op == "linear":
        if not state["case"]["train"]:
            with torch.no_grad():
                return {"y": nnops.linear_act(state["x"], state["w"], state["b"], state["r"], activation=state["case"]["act"])}
        leaves = [state[key] for key in ("x", "w", "b", "r") if state[key] is not None]
        y = nnops.linear_act(state["x"], state["w"], state["b"], state["r"], activation=state["case"]["act"])
        grads = torch.autograd.grad(y, leaves, state["dy"])
        return dict(zip(("y", "dx", "dw", "db", "dr"), (y.detach(),) + grads))
    if op == "ce":
        leaves = [state[key] for key in ("x", "w", "b") if state[key] is not None]
        loss = nnops.linear_cross_entropy(state["x"], state["w"], state["t"], bias=state["b"], class_weight=state["cw"])
        grads = torch.autograd.grad(loss, leaves)
        return dict(zip(("loss", "dx", "dw", "db"), (loss.detach(),) + grads))
    norm = nnops.clip_grad_norm_(state["grads"], MAX_NORM, out=state["out"])
    return {"norm": norm, "out": state["flat"]}


def work(case):
    """each input read once and each output written once; the products that the formulas cannot do without"""
    if case["op"] == "linear":
        m, k, n, e = case["rows"], case["k"], case["n"], SIZE[case["dtype"]]
        elems = m * k + n * k + n + m * n * (2 if case["residual"] else 1)
        flops = 2 * m * n * k
        if case["train"]:
            elems += m * n + m * k + n * k + n
            flops *= 3
        return {"bytes": elems * e, "flops": flops}
    if case["op"] == "ce":
        m, k, v, e = case["rows"], case["k"], case["classes"], SIZE[case["dtype"]]
        elems = 2 * (m * k + v * k + (v if case["bias"] else 0))
        return {"bytes": elems * e + 8 * m + (4 * v if case["weighted"] else 0), "flops": 6 * m * k * v}
    return {"bytes": case["elements"] * (SIZE[case["dtype"]] + SIZE[case["out_dtype"]]), "flops": 3 * case["elements"]}


def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "linear":
        x, w, b = (st[key].detach().to(f64) for key in ("x", "w", "b"))
        z = torch.addmm(b, x, w.T)
        cdf = torch.special.ndtr(z) if case["act"] == "gelu" else torch.sigmoid(z)
        y = {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, torch.zeros_like(z)), "gelu": lambda: z * cdf, "silu": lambda: z * cdf}[case["act"]]()
        if st["r"] is not None:
            y = y + st["r"].detach().to(f64)
        if not case["train"]:
            return {"y": y}
        dy = st["dy"].to(f64)
        slope = {"none": lambda: torch.ones_like(z), "relu": lambda: torch.heaviside(z, torch.zeros_like(z)),
                 "gelu": lambda: cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), "silu": lambda: cdf + z * cdf * (1 - cdf)}[case["act"]]()
        dz = slope * dy
        out = {"y": y, "dx": torch.mm(dz, w), "dw": torch.mm(dz.T.contiguous(), x), "db": dz.sum(dim=0)}
        if st["r"] is not None:
            out["dr"] = dy
        return out
    if case["op"] == "ce":
        x, w = st["x"].detach().to(f64), st["w"].detach().to(f64)
        b = st["b"].detach().to(f64) if st["b"] is not None else torch.zeros(w.shape[0], dtype=f64, device="cuda")
        out_dx, out_dw, out_db, loss = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b), 0.0
        rows = torch.nonzero(st["t"] != -100).squeeze(1)
        weight = torch.ones(w.shape[0], dtype=f64, device="cuda") if st["cw"] is None else st["cw"].to(f64)
        total = weight[st["t"][rows]].sum()
        for part in rows.split(4096):        # pieces of the rows: the 64-bit logits of all of them are large
            t = st["t"][part]
            logp = torch.log_softmax(torch.addmm(b, x[part], w.T), dim=1)
            share = weight[t] / total
            loss = loss - (logp[torch.arange(len(part), device="cuda"), t] * share).sum()
            p = logp.exp_()
            p[torch.arange(len(part), device="cuda"), t] -= 1.0
            p *= share[:, None]
            out_dx[part] = p @ w
            out_dw += p.T.contiguous() @ x[part]
            out_db += p.sum(dim=0)
        out = {"loss": loss, "dx": out_dx, "dw": out_dw}
        if st["b"] is not None:
            out["db"] = out_db
        return out
    norm = math.sqrt(sum(float((g.to(f64) ** 2).sum()) for g in st["grads"]))
    factor = min(1.0, MAX_NORM / (norm + 1e-6))
    return {"norm": torch.tensor(norm, dtype=f64, device="cuda"), "out": torch.cat([g.to(f64) for g in st["grads"]]) * factor}
