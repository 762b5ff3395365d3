"""The semantic head's operators, as they are measured: what a pass computes, on which sizes, and its plain form.

Two operators of the semantic path (per-Gaussian features rendered to a [H,W,D] plane, a small head that turns the plane
into class scores, a segmentation teacher whose top scores per pixel train it):

* ``linear``   y = act(x W^T + b) + r, one layer of the head, and its backward pass (``ops.linear_act``);
* ``distill``  the temperature-softened divergence between a teacher's top-K scores and the student's softmax over all V
  classes, and its gradient (``losses.topk_distill_loss``).

Frame sizes are those of the framework's own workloads: 128x128, 800x800, 1280x720 and 1920x1080 pixels.
"""
import math

import torch

own = False

_T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_IDX = {"i32": torch.int32, "i64": torch.int64}


def _lin(name, rows, k, n, dtype, act, bias=True, res=False, pitch=0, train=False):
    """``pitch``: extra columns between the rows of x (the plane is a slice of a wider render)."""
    return dict(name=name, op="linear", rows=rows, k=k, n=n, dtype=dtype, act=act, bias=bias, res=res, pitch=pitch,
                train=train)


def _dis(name, rows, v, k, dtype, tdtype, idx, reduction="mean", weight=False, temperature=1.0, train=True):
    return dict(name=name, op="distill", rows=rows, v=v, k=k, dtype=dtype, tdtype=tdtype, idx=idx, reduction=reduction,
                weight=weight, temperature=temperature, train=train)


def listed():
    return [
        # one picked point's feature to its class scores: pure latency
        _lin("linear_pick_f32", 1, 64, 150, "f32", "none"),
        # first layer on a 128x128 frame; the features are the leading channels of a render that carries depth behind them
        _lin("linear_frame128_f32", 16384, 32, 64, "f32", "relu", pitch=1),
        # widening layer on an 800x800 frame in half-width storage
        _lin("linear_frame800_bf16", 640000, 64, 128, "bf16", "gelu"),
        # residual block on a 1280x720 frame in full precision
        _lin("linear_frame720_f32", 921600, 64, 64, "f32", "silu", res=True),
        # class layer, one training step on an 800x800 frame
        _lin("linear_train_classes_f32", 640000, 32, 150, "f32", "none", train=True),
        # residual block, one training step on an 800x800 frame
        _lin("linear_train_block_bf16", 640000, 128, 128, "bf16", "gelu", res=True, train=True),
        # projection to a wide language-aligned embedding with odd sizes throughout
        _lin("linear_train_wide_f16", 100003, 513, 768, "f16", "relu", bias=False, train=True),
        # one picked point's loss and gradient: latency
        _dis("distill_pick_f32", 1, 150, 8, "f32", "f32", "i64"),
        # one training step on an 800x800 frame, teacher record kept in half width
        _dis("distill_frame800_f32", 640000, 150, 16, "f32", "f16", "i32", temperature=2.0),
        # long-tailed vocabulary on a quarter-size 1280x720 frame, odd class count, confidence-weighted pixels
        _dis("distill_open_bf16", 230400, 1203, 32, "bf16", "f16", "i64", weight=True),
        # open vocabulary as large as a language model's, a batch of sampled pixels, per-row losses
        _dis("distill_vocab_f16", 4099, 32003, 64, "f16", "f16", "i64", reduction="none", temperature=1.5),
        # per-pixel loss map of a 1920x1080 validation frame with few classes
        _dis("distill_eval1080_bf16", 2073600, 21, 4, "bf16", "bf16", "i32", reduction="none", weight=True, train=False),
    ]


def _cost(case):
    """Rough time of a pass on the card, to keep drawn cases below the largest listed one."""
    w = work(case)
    rate = 80e12 if case["dtype"] == "f32" else 500e12
    return w["bytes"] / 4e12 + w["flops"] / rate


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        dtype = rng.choice(["f32", "bf16", "f16"])
        train = rng.random() < 0.6
        if rng.random() < 0.5:
            case = _lin("", _log(rng, 1, 2073600), _log(rng, 3, 1024), _log(rng, 2, 1500), dtype,
                        rng.choice(["none", "relu", "gelu", "silu"]), bias=rng.random() < 0.7, res=rng.random() < 0.4,
                        pitch=rng.choice([0, 0, 1, 4]), train=train)
            elements = case["rows"] * max(case["k"], case["n"])
        else:
            v = _log(rng, 2, 32768)
            case = _dis("", _log(rng, 1, 2073600), v, min(v, _log(rng, 1, 64)), dtype, rng.choice(["f32", "bf16", "f16"]),
                        rng.choice(["i32", "i64"]), reduction=rng.choice(["mean", "sum", "none"]) if train else "none",
                        weight=rng.random() < 0.5, temperature=rng.choice([0.5, 1.0, 2.0]), train=train)
            elements = case["rows"] * v
        if elements <= 300_000_000 and _cost(case) <= top:
            del case["name"]
            return case


def work(case):
    e = _SIZE[case["dtype"]]
    r = case["rows"]
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        bias = n if case["bias"] else 0
        b = r * k + n * k + bias + r * n * (2 if case["res"] else 1)
        if case["train"]:  # and the upstream gradient in, the gradients of x, W and b out
            b += r * n + r * k + n * k + bias
        return {"bytes": e * b, "flops": 2 * r * n * k * (3 if case["train"] else 1)}
    v, k = case["v"], case["k"]
    idx = 4 if case["idx"] == "i32" else 8
    out = 4 * (r if case["reduction"] == "none" else 1)
    b = r * v * e + r * k * (idx + _SIZE[case["tdtype"]]) + (4 * r if case["weight"] else 0) + out
    if case["train"]:
        b += r * v * e + (4 * r if case["reduction"] == "none" else 0)
    return {"bytes": b, "flops": r * v * (8 if case["train"] else 4)}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    dt, r = _T[case["dtype"]], case["rows"]
    st = dict(case=case)
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        x = randn(r, k + case["pitch"])
        # pixels that no Gaussian covers: a zero feature row
        x[torch.rand(r, generator=g, device=dev) < 0.1] = 0.0
        st["x"] = x.to(dt)[:, :k]
        bound = 1.0 / math.sqrt(k)
        st["w"] = ((torch.rand(n, k, generator=g, device=dev) * 2 - 1) * bound).to(dt)
        st["b"] = ((torch.rand(n, generator=g, device=dev) * 2 - 1) * bound).to(dt) if case["bias"] else None
        st["res"] = randn(r, n).to(dt) if case["res"] else None
        if case["train"]:
            st["dy"] = randn(r, n).to(dt)
            for key in ("x", "w", "b", "res"):
                if st[key] is not None:
                    st[key] = st[key].detach().requires_grad_(True)
        return st
    v, k = case["v"], case["k"]
    teacher = randn(r, v).mul_(3.0)
    top, idx = teacher.topk(k, dim=-1)
    st["logits"] = teacher.mul_(0.5).add_(randn(r, v)).to(dt)
    del teacher
    # the teacher's list ends where its scores get negligible: 1 .. K entries; every tenth pixel has none at all
    kept = torch.randint(1, k + 1, (r, 1), generator=g, device=dev)
    kept[torch.rand(r, 1, generator=g, device=dev) < 0.1] = 0
    if r == 1:
        kept.fill_(k)
    gone = torch.arange(k, device=dev)[None] >= kept
    st["idx"] = idx.masked_fill(gone, -1).to(_IDX[case["idx"]])
    st["top"] = top.masked_fill(gone, 0.0).to(_T[case["tdtype"]])
    st["weight"] = torch.rand(r, generator=g, device=dev) if case["weight"] else None
    if case["train"]:
        st["logits"].requires_grad_(True)
        st["g"] = torch.rand(r, generator=g, device=dev) if case["reduction"] == "none" else torch.ones((), device=dev)
    return st


# ---- plain forms ------------------------------------------------------------------------------------------------
def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _linear_plain(st):
    case = st["case"]
    dt = _T[case["dtype"]]
    x, w = st["x"].detach().float(), st["w"].detach().float()
    z = x @ w.t()
    if st["b"] is not None:
        z = z + st["b"].detach().float()
    y = _act(z, case["act"])
    if st["res"] is not None:
        y = y + st["res"].detach().float()
    out = {"y": y.to(dt)}
    if case["train"]:
        dz = st["dy"].float() * _act_slope(z, case["act"])
        out["dx"] = (dz @ w).to(dt)
        out["dw"] = (dz.t() @ x).to(dt)
        if st["b"] is not None:
            out["db"] = dz.sum(0).to(dt)
        if st["res"] is not None:
            out["dres"] = st["dy"]
    return out


def _distill_plain(st):
    case = st["case"]
    T = case["temperature"]
    s = st["logits"].detach().float() / T
    v = s.shape[-1]
    m = s.max(dim=-1, keepdim=True).values
    e = torch.exp(s - m)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total) + m
    idx = st["idx"].long()
    there = (idx >= 0) & (idx < v)
    at = torch.where(there, idx, torch.zeros_like(idx))
    u = torch.where(there, st["top"].float() / T, torch.full_like(st["top"], -math.inf, dtype=torch.float32))
    um = u.max(dim=-1, keepdim=True).values
    um = torch.where(um > -math.inf, um, torch.zeros_like(um))
    pe = torch.exp(u - um)
    pt = pe.sum(-1, keepdim=True)
    alive = pt > 0
    pt = torch.where(alive, pt, torch.ones_like(pt))
    p = pe / pt
    log_p = u - um - torch.log(pt)
    log_q = torch.gather(s, -1, at) - log_total
    term = torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p))
    row = (T * T) * term.sum(-1)
    w = alive[:, 0].float()
    if st["weight"] is not None:
        w = w * st["weight"]
    row = row * w
    if case["reduction"] == "none":
        loss, coef = row, w
    else:
        total_w = w.double().sum().float()
        loss = row.double().sum().float()
        coef = w
        if case["reduction"] == "mean":
            total_w = torch.where(total_w > 0, total_w, torch.ones_like(total_w))
            loss, coef = loss / total_w, w / total_w
    if not case["train"]:
        return {"loss": loss}
    grad = e.div_(total)
    grad.scatter_add_(-1, at, -p)
    grad.mul_((T * coef * st["g"])[:, None])
    return {"loss": loss, "dlogits": grad.to(_T[case["dtype"]])}


def run(state):
    case = state["case"]
    if not own:
        return _linear_plain(state) if case["op"] == "linear" else _distill_plain(state)
    if case["op"] == "linear":
        from fusionsense_amd import ops
        y = ops.linear_act(state["x"], state["w"], state["b"], act=case["act"], residual=state["res"])
        if not case["train"]:
            return {"y": y}
        names = [k for k in ("x", "w", "b", "res") if state[k] is not None]
        grads = torch.autograd.grad(y, [state[k] for k in names], state["dy"])
        return {"y": y.detach(), **{"d" + k: v for k, v in zip(names, grads)}}
    from fusionsense_amd import losses
    loss = losses.topk_distill_loss(state["logits"], state["idx"], state["top"], temperature=case["temperature"],
                                    weight=state["weight"], reduction=case["reduction"])
    if not case["train"]:
        return {"loss": loss}
    grad, = torch.autograd.grad(loss, [state["logits"]], state["g"])
    return {"loss": loss.detach(), "dlogits": grad}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "linear":
        x, w = st["x"].detach().double().requires_grad_(True), st["w"].detach().double().requires_grad_(True)
        leaves = {"x": x, "w": w}
        z = torch.matmul(x, w.transpose(0, 1))
        if st["b"] is not None:
            leaves["b"] = st["b"].detach().double().requires_grad_(True)
            z = z + leaves["b"][None, :]
        y = {"none": lambda t: t, "relu": torch.relu, "gelu": torch.nn.functional.gelu,
             "silu": torch.nn.functional.silu}[case["act"]](z)
        if st["res"] is not None:
            leaves["res"] = st["res"].detach().double().requires_grad_(True)
            y = y + leaves["res"]
        if not case["train"]:
            return {"y": y.detach()}
        grads = torch.autograd.grad(y, list(leaves.values()), st["dy"].double())
        return {"y": y.detach(), **{"d" + k: v for k, v in zip(leaves, grads)}}
    T = float(case["temperature"])
    s = st["logits"].detach().double()
    idx, v = st["idx"].long(), case["v"]
    pad = torch.logical_or(idx < 0, idx >= v)
    has = ~pad.all(-1)
    log_p = torch.log_softmax((st["top"].double() / T).masked_fill(pad, -math.inf), -1)
    log_p = log_p.masked_fill(pad, -math.inf)
    p = log_p.exp()
    log_q = torch.log_softmax(s / T, -1)
    picked = torch.gather(log_q, -1, idx.masked_fill(pad, 0))
    kl = (p * (log_p.masked_fill(pad, 0.0) - picked)).sum(-1) * T * T
    w = has.double() if st["weight"] is None else has.double() * st["weight"].double()
    scale = {"none": 1.0, "sum": 1.0, "mean": 1.0 / max(float(w.sum()), 1e-300) if float(w.sum()) > 0 else 1.0}
    scale = scale[case["reduction"]]
    loss = kl * w * scale if case["reduction"] == "none" else (kl * w).sum() * scale
    if not case["train"]:
        return {"loss": loss}
    target = torch.zeros_like(log_q).scatter_add_(-1, idx.masked_fill(pad, 0), p)
    grad = (log_q.exp() - target) * (T * scale * w * st["g"].double())[:, None]
    return {"loss": loss, "dlogits": grad}
