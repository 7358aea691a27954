"""The classification head's operators and the matrix update, as they are measured: what is called, on what, and the same in
plain torch operations.

    loss    softmax cross entropy of a linear head over V classes, logits not kept, and its gradients
    answer  expected bin centre under the same head's softmax, and its gradients
    update  an update matrix orthogonalised by Newton-Schulz products

`run` with `own` false is the plain form; with `own` true it makes the calls a program makes of this package.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
IGNORE = -100
LARGEST = 8192 * 65536 * 1024        # rows x classes x features of the largest head
LARGEST_UPDATE = 4096 ** 3


def listed():
    return [
        # the head of a depth network at cost-volume resolution (96x320, 80 bins), 12 targets, supervised by a sparse laser
        # scan: one pixel in twenty has a depth
        dict(name="loss_bins_sparse_bf16", kind="loss", rows=12 * 96 * 320, features=64, classes=80, type="bfloat16",
             keep=0.05, reduction="mean", train=True),
        # the same head in float32 on dense synthetic depth, two targets
        dict(name="loss_bins_dense_f32", kind="loss", rows=2 * 96 * 320, features=64, classes=80, type="float32",
             keep=1.0, reduction="mean", train=True),
        # a training step over a large vocabulary
        dict(name="loss_vocab_bf16", kind="loss", rows=8192, features=1024, classes=65536, type="bfloat16", keep=1.0,
             reduction="mean", train=True),
        # odd sizes, a ragged batch with padding, and a weight for every row
        dict(name="loss_vocab_odd_f16", kind="loss", rows=1003, features=771, classes=50021, type="float16", keep=0.7,
             reduction="none", train=True),
        # one position answered from a bin head: latency
        dict(name="answer_one_row_f32", kind="answer", rows=1, features=256, classes=80, type="float32", train=False),
        # one row over a large table: the table is read once
        dict(name="answer_one_row_wide_bf16", kind="answer", rows=1, features=1024, classes=65536, type="bfloat16",
             train=False),
        # a batch of depth maps predicted from its features
        dict(name="answer_maps_bf16", kind="answer", rows=12 * 96 * 320, features=64, classes=80, type="bfloat16",
             train=False),
        # the same answer trained through: its gradient reaches features and weights
        dict(name="answer_maps_train_bf16", kind="answer", rows=2 * 96 * 320, features=128, classes=256, type="bfloat16",
             train=True),
        # the first convolution of a network (64 filters of 3x7x7): latency
        dict(name="update_64x147_f32", kind="update", batch=1, m=64, n=147, type="float32", steps=5),
        # a late convolution (512 filters of 512x3x3)
        dict(name="update_512x4608_f32", kind="update", batch=1, m=512, n=4608, type="float32", steps=5),
        # a large square layer
        dict(name="update_4096_bf16", kind="update", batch=1, m=4096, n=4096, type="bfloat16", steps=5),
        # a stack of tall matrices of odd size
        dict(name="update_tall_stack_f32", kind="update", batch=4, m=1531, n=510, type="float32", steps=5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["loss", "answer", "update"])
    t = rng.choice(sorted(TYPES))
    if kind == "update":
        while True:
            c = dict(kind=kind, batch=rng.choice([1, 1, 2, 5]), m=_log(rng, 8, 8192), n=_log(rng, 8, 8192), type=t, steps=5)
            s, l = sorted((c["m"], c["n"]))
            if c["batch"] * s * s * l <= LARGEST_UPDATE // 4:
                return c
    while True:
        if rng.random() < 0.5:    # bins of a map
            c = dict(kind=kind, rows=_log(rng, 1, 12 * 96 * 320), features=_log(rng, 16, 256), classes=_log(rng, 2, 512))
        else:                     # a vocabulary
            c = dict(kind=kind, rows=_log(rng, 1, 8192), features=_log(rng, 32, 2048), classes=_log(rng, 512, 100000))
        if c["rows"] * c["features"] * c["classes"] <= LARGEST // 8:
            break
    if rng.random() < 0.6:
        c["features"] = -(-c["features"] // 8) * 8
    c.update(type=t, train=rng.random() < 0.7)
    if kind == "loss":
        c.update(keep=rng.choice([1.0, 1.0, 0.8, 0.05]), reduction=rng.choice(["mean", "sum", "none"]))
    return c


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if case["kind"] == "update":
        b, m, n = case["batch"], case["m"], case["n"]
        r = max(1, min(m, n) // 16)       # a gradient averaged over steps: a few strong directions over noise
        strong = torch.matmul(normal(b, m, r), normal(b, r, n))
        return dict(case=case, update=((strong / math.sqrt(r) + normal(b, m, n)) * 1e-3).to(t))
    rows, d, v = case["rows"], case["features"], case["classes"]
    weight = normal(v, d) / math.sqrt(d)
    targets = torch.randint(0, v, (rows,), generator=g, device=DEV)
    # features that have learned something of their class: its logit stands out by a few units
    hidden = normal(rows, d) + 3.0 * weight[targets]
    state = dict(case=case, hidden=hidden.to(t), weight=weight.to(t))
    if case["kind"] == "loss":
        drop = torch.rand(rows, generator=g, device=DEV) >= case["keep"]
        drop[0] = False
        state["targets"] = torch.where(drop, torch.full_like(targets, IGNORE), targets)
    else:                                 # bins spaced as the plane sweep's: finer near the camera, up to 80 m
        i = torch.arange(v, device=DEV, dtype=torch.float64)
        state["centers"] = ((torch.exp((i + 1) * math.log(2) / v) - 1) * 80).float()
    state["upstream"] = torch.rand(rows, generator=g, device=DEV) + 0.5
    if case["train"]:
        state["hidden"].requires_grad_(True)
        state["weight"].requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------------------- the package's calls
def _run_own(state):
    from depth_estimation_amd import metrics, optim, synthesis
    case = state["case"]
    if case["kind"] == "update":
        return optim.orthogonalize(state["update"], steps=case["steps"], coefficients=COEFFICIENTS, eps=EPS)
    hidden, weight = state["hidden"], state["weight"]
    if case["kind"] == "loss":
        out = metrics.linear_cross_entropy(hidden, weight, state["targets"], ignore_index=IGNORE,
                                           reduction=case["reduction"])
        up = state["upstream"] if case["reduction"] == "none" else None
    else:
        out = synthesis.depth_from_bins(hidden, weight, state["centers"])
        up = state["upstream"]
    if not case["train"]:
        return {"out": out}
    gh, gw = torch.autograd.grad(out, (hidden, weight), up)
    return {"out": out.detach(), "g_hidden": gh, "g_weight": gw}


# ------------------------------------------------------------------------------------------------------ the plain form
def _plain_loss(state):
    case = state["case"]
    hidden, weight, targets = state["hidden"].detach(), state["weight"].detach(), state["targets"]
    kept = (targets != IGNORE).nonzero()[:, 0]
    h, w, t = hidden[kept].float(), weight.float(), targets[kept]
    logits = h @ w.t()
    top = logits.max(dim=1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(dim=1, keepdim=True)
    each = (torch.log(total) + top)[:, 0] - logits.gather(1, t[:, None])[:, 0]
    if case["reduction"] == "none":
        out = torch.zeros(targets.shape[0], device=DEV).index_copy(0, kept, each)
        up = state["upstream"][kept]
    else:
        out = each.sum() if case["reduction"] == "sum" else each.sum() / kept.shape[0]
        up = torch.full_like(each, 1.0 if case["reduction"] == "sum" else 1.0 / kept.shape[0])
    if not case["train"]:
        return {"out": out}
    p = e / total
    p.scatter_add_(1, t[:, None], torch.full_like(p[:, :1], -1.0))
    p *= up[:, None]
    gh = torch.zeros_like(hidden).index_copy(0, kept, (p @ w).to(hidden.dtype))
    return {"out": out, "g_hidden": gh, "g_weight": (p.t() @ h).to(weight.dtype)}


def _plain_answer(state):
    hidden, weight, c = state["hidden"].detach(), state["weight"].detach(), state["centers"]
    h, w = hidden.float(), weight.float()
    logits = h @ w.t()
    e = torch.exp(logits - logits.max(dim=1, keepdim=True).values)
    p = e / e.sum(dim=1, keepdim=True)
    out = (p * c).sum(dim=1)
    if not state["case"]["train"]:
        return {"out": out}
    dl = p * (c - out[:, None]) * state["upstream"][:, None]
    return {"out": out, "g_hidden": (dl @ w).to(hidden.dtype), "g_weight": (dl.t() @ h).to(weight.dtype)}


def _plain_update(state):
    u = state["update"]
    a, b, c = COEFFICIENTS
    x = u.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1).contiguous()
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + EPS)
    for _ in range(state["case"]["steps"]):
        s = torch.matmul(x, x.transpose(-2, -1).contiguous())
        x = a * x + torch.matmul(b * s + c * torch.matmul(s, s), x)
    return (x.transpose(-2, -1).contiguous() if tall else x).to(u.dtype)


def run(state):
    if own:
        return _run_own(state)
    return {"loss": _plain_loss, "answer": _plain_answer, "update": _plain_update}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "update":
        done = []
        for u in state["update"].double():
            # on the singular values: X = U f(S) V^T, f the composed polynomial; U and V from the smaller Gram matrix would
            # square the condition, so the products are formed
            z = u / (torch.linalg.vector_norm(u) + EPS)
            side = z.shape[0] <= z.shape[1]
            for _ in range(case["steps"]):
                gram = z @ z.mT if side else z.mT @ z
                poly = COEFFICIENTS[1] * gram + COEFFICIENTS[2] * (gram @ gram)
                poly.diagonal().add_(COEFFICIENTS[0])
                z = poly @ z if side else z @ poly
            done.append(z)
        return torch.stack(done)
    with torch.no_grad():
        h, w = state["hidden"].double(), state["weight"].double()
        outs, ghs, gw = [], [], torch.zeros_like(w)
        loss = case["kind"] == "loss"
        n = h.shape[0]
        if loss:
            valid = state["targets"] != IGNORE
            count = valid.sum().double()
            up = {"none": state["upstream"].double(), "sum": torch.ones(n, device=DEV, dtype=torch.float64),
                  "mean": torch.ones(n, device=DEV, dtype=torch.float64) / count}[case["reduction"]]
        else:
            up, c = state["upstream"].double(), state["centers"].double()
        for lo in range(0, n, 16384):
            hs, us = h[lo:lo + 16384], up[lo:lo + 16384]
            logp = torch.log_softmax(hs @ w.mT, dim=1)
            p = logp.exp()
            if loss:
                ok, t = valid[lo:lo + 16384], state["targets"][lo:lo + 16384].clamp(min=0)
                outs.append(torch.where(ok, -logp[torch.arange(len(t), device=DEV), t], 0.0))
                p[torch.arange(len(t), device=DEV), t] -= 1.0
                p *= torch.where(ok, us, 0.0)[:, None]
            else:
                mean = p @ c
                outs.append(mean)
                p *= us[:, None] * (c[None, :] - mean[:, None])
            if case["train"]:
                ghs.append(p @ w)
                gw += p.mT @ hs
        out = torch.cat(outs)
        if loss and case["reduction"] != "none":
            out = out.sum() / (count if case["reduction"] == "mean" else 1.0)
        return {"out": out, "g_hidden": torch.cat(ghs), "g_weight": gw} if case["train"] else {"out": out}


def work(case):
    e = 4 if case["type"] == "float32" else 2
    if case["kind"] == "update":
        b, (s, l) = case["batch"], sorted((case["m"], case["n"]))
        # two symmetric products (half of them) and a full one a step
        return {"bytes": 2 * e * b * s * l, "flops": case["steps"] * b * (s * s * l + s ** 3 + 2 * s * s * l)}
    n, d, v = case["rows"], case["features"], case["classes"]
    kept = n if case["kind"] == "answer" else max(1, round(n * case["keep"]))
    nbytes = e * (kept * d + v * d) + (4 * v + 4 * n if case["kind"] == "answer" else 8 * n + 4)
    flops = 2 * kept * d * v
    if case["train"]:
        nbytes += e * (n * d + v * d) + 4 * n
        flops *= 3
    return {"bytes": nbytes, "flops": flops}
