"""The two ends of a language model measured next to their plain forms: the embedding lookup and its gradient, and
the last linear layer with its loss, cross entropy or distillation from a teacher's top logits, without the logits.

Every case is one call a program makes (a "train" case the forward and the backward call of one step).  Token rows are
[batch, tokens, width], f32 (the embedding also f64).  `own` False runs the plain form, elementary torch operations;
`own` True runs the calls of this package.
"""
import math

import torch

own = False

DEVICE = "cuda"


# ---- cases --------------------------------------------------------------------


def listed():
    return [
        # the next token of each of 16 sequences looked up: a generation step, where the time to issue the call counts
        _embedding("embedding_one_token", 16, 1, 32000, 1024),
        # a prompt of 4 x 4096 tokens, with the scale of tables that are shared with the last layer
        _embedding("embedding_prompt", 4, 4096, 50000, 2048),
        # the gradient of a training batch in full, a few tokens of padding at each end
        _embedding("embedding_backward", 8, 2048, 50000, 1024, padding=0.05, direction="backward"),
        # forward and gradient of a small odd table kept in 64 bits, added to the gradient that is there
        _embedding("embedding_train_f64", 3, 777, 5003, 203, padding=0.05, direction="train", dtype="f64",
                   accumulate=True),
        # one candidate token of each of 4 sequences scored
        _ce("cross_entropy_few_tokens", 4, 1, 32000, 1024),
        # the answer part of a prompt scored
        _ce("cross_entropy_score", 1, 500, 32000, 768, masked=0.3),
        # a training step whose sizes fit nothing: smoothed targets, a third of the rows masked
        _ce("cross_entropy_train_odd", 3, 333, 10007, 521, masked=0.35, smoothing=0.1, direction="train"),
        # the largest training step
        _ce("cross_entropy_train", 4, 2048, 50000, 2048, direction="train"),
        # a step on the few positions at which a draft was refused
        _distill("distillation_few_tokens", 7, 1, 32000, 1024, 32, 1.0, direction="train"),
        # a student held against its teacher's kept logits
        _distill("distillation_score", 2, 1024, 32000, 1024, 50, 2.0, masked=0.1),
        # a training step whose sizes fit nothing, rows and entries of padding
        _distill("distillation_train_odd", 2, 511, 12345, 330, 17, 1.5, masked=0.2, direction="train"),
        # a training step on a teacher's 64 largest logits per position
        _distill("distillation_train", 4, 1024, 32000, 2048, 64, 2.0, direction="train"),
    ]


def _embedding(name, B, T, V, D, padding=0.0, direction="forward", dtype="f32", accumulate=False):
    return {"name": name, "op": "embedding", "direction": direction, "B": B, "T": T, "V": V, "D": D,
            "padding": padding, "dtype": dtype, "accumulate": accumulate}


def _ce(name, B, T, V, D, masked=0.0, smoothing=0.0, direction="forward"):
    return {"name": name, "op": "cross_entropy", "direction": direction, "B": B, "T": T, "V": V, "D": D,
            "masked": masked, "smoothing": smoothing}


def _distill(name, B, T, V, D, K, temperature, masked=0.0, direction="forward"):
    return {"name": name, "op": "distillation", "direction": direction, "B": B, "T": T, "V": V, "D": D, "K": K,
            "temperature": temperature, "masked": masked}


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embedding", "cross_entropy", "cross_entropy", "distillation"])
    V = _spread(rng, 300, 130000)
    D = rng.choice([_spread(rng, 16, 4096), 8 * _spread(rng, 2, 512), 64 * rng.randint(1, 64)])
    B, T = rng.randint(1, 16), rng.choice([1, _spread(rng, 1, 4096), _spread(rng, 64, 4096)])
    if op == "embedding":
        while B * T * D > 4 * 4096 * 2048 or V * D > 1 << 27:
            T, V = max(1, T // 2), max(300, V // 2 + 1)
        return _unnamed(_embedding("", B, T, V, D, padding=rng.choice([0.0, 0.1]),
                                   direction=rng.choice(["forward", "backward", "train"]),
                                   dtype=rng.choice(["f32", "f32", "f64"]), accumulate=rng.random() < 0.4))
    while B * T * V * D > 8192 * 50000 * 2048 or V * D > 1 << 28 or B * T * V > 8192 * 50000:
        if B * T > 1024 or V < 600:
            B, T = max(1, B // 2), max(1, T - T // 4)
        else:
            V = V // 2 + 1
    direction = rng.choice(["forward", "train", "train"])
    masked = rng.choice([0.0, 0.0, 0.2, 0.7])
    if op == "cross_entropy":
        return _unnamed(_ce("", B, T, V, D, masked, rng.choice([0.0, 0.0, 0.1]), direction))
    return _unnamed(_distill("", B, T, V, D, rng.randint(1, 128), rng.choice([1.0, 2.0, 3.5]), masked, direction))


def _unnamed(c):
    del c["name"]
    return c


# ---- inputs -------------------------------------------------------------------


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    B, T, V, D = c["B"], c["T"], c["V"], c["D"]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device=DEVICE, dtype=torch.float64)

    def tokens(*shape):  # a few tokens make up most of a text: the r-th most frequent comes with a share of 1 / r
        rank = (V ** uniform(*shape)).long().clamp(1, V) - 1
        return torch.randperm(V, generator=g, device=DEVICE)[rank]

    if c["op"] == "embedding":
        dt = torch.float64 if c["dtype"] == "f64" else torch.float32
        ids = tokens(B, T)
        ids[uniform(B, T) < c["padding"]] = -1
        s = {"case": c, "ids": ids, "scale": math.sqrt(D)}
        if c["direction"] != "backward":
            s["table"] = normal(V, D, dtype=dt) / math.sqrt(D)
        if c["direction"] != "forward":
            s["grad"] = normal(B, T, D, dtype=dt)
            if c["accumulate"]:
                s["before"] = normal(V, D, dtype=dt)
        return s
    # states as a last norm leaves them; the token that was taken is the likelier one for having been trained on
    weight = normal(V, D) * (2.0 / math.sqrt(D))
    target = tokens(B, T)
    hidden = normal(B, T, D) + weight[target] * 1.5
    absent = uniform(B, T) < c["masked"]
    s = {"case": c, "hidden": hidden, "weight": weight}
    if c["op"] == "cross_entropy":
        s["targets"] = torch.where(absent, -100, target)
    else:
        K = min(c["K"], V)
        s["ids"] = torch.stack([(target + k * (1 + (target + k) % 7)) % V for k in range(K)], -1)
        z = normal(B, T, K) * 2.0
        z[..., 0] += 3.0
        z, _ = z.sort(-1, descending=True)
        s["ids"][uniform(B, T, K) < 0.02] = -1  # padding among the entries
        s["ids"][absent] = -1
        s["logits"] = z
    if c["direction"] == "train":
        s["grad"] = torch.rand((B, T), generator=g, device=DEVICE) / max(1, B * T)
    return s


# ---- one pass -------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from tensorrs_b200 import device as trs

    c = s["case"]
    if c["op"] == "embedding":
        ids = trs.view_of(s["ids"])
        out = gt = None
        if c["direction"] != "backward":
            out = torch.empty((c["B"], c["T"], c["D"]), device=DEVICE, dtype=s["table"].dtype)
            trs.embedding(trs.view_of(s["table"]), ids, s["scale"], out)
        if c["direction"] != "forward":
            acc = c["accumulate"]
            gt = s["before"].clone() if acc else torch.empty((c["V"], c["D"]), device=DEVICE, dtype=s["grad"].dtype)
            trs.embedding_backward(trs.view_of(s["grad"]), ids, s["scale"], gt, accumulate=acc)
        return tuple(t for t in (out, gt) if t is not None)
    h, w = trs.view_of(s["hidden"]), trs.view_of(s["weight"])
    loss, lse = torch.empty((c["B"], c["T"]), device=DEVICE), torch.empty((c["B"], c["T"]), device=DEVICE)
    if c["op"] == "cross_entropy":
        t = trs.view_of(s["targets"])
        trs.linear_cross_entropy(h, w, t, loss, lse, smoothing=c["smoothing"])
    else:
        ids, z = trs.view_of(s["ids"]), trs.view_of(s["logits"])
        trs.linear_distillation(h, w, ids, z, c["temperature"], loss, lse)
    if c["direction"] == "forward":
        return loss, lse
    dh, dw = torch.empty_like(s["hidden"]), torch.empty_like(s["weight"])
    g, l = trs.view_of(s["grad"]), trs.view_of(lse)
    if c["op"] == "cross_entropy":
        trs.linear_cross_entropy_backward(g, h, w, t, l, dh, dw, smoothing=c["smoothing"])
    else:
        trs.linear_distillation_backward(g, h, w, ids, z, l, c["temperature"], dh, dw)
    return loss, lse, dh, dw


def _run_plain(s):
    c = s["case"]
    if c["op"] == "embedding":
        return _plain_embedding(s)
    B, T, V, D = c["B"], c["T"], c["V"], c["D"]
    temp = c.get("temperature", 1.0)
    if c["op"] == "cross_entropy":
        t = s["targets"].reshape(-1, 1)
        there = (t >= 0) & (t < V)
        t = torch.where(there, t, 0)
        p = there * (1.0 - c["smoothing"])
        ln_p = 0.0
    else:
        t = s["ids"].reshape(B * T, -1)
        there = (t >= 0) & (t < V)
        t = torch.where(there, t, 0)
        z = (s["logits"].reshape(B * T, -1) / temp).masked_fill(~there, -math.inf)
        top = z.amax(-1, keepdim=True)
        e = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = e.sum(-1, keepdim=True)
        total = torch.where(total == 0, torch.ones_like(total), total)
        p = e / total
        ln_p = torch.where(p > 0, z - top - torch.log(total), torch.zeros_like(z))
    live = there.any(-1, keepdim=True)
    h = torch.where(live, s["hidden"].reshape(B * T, D), 0.0)
    x = torch.matmul(h, s["weight"].T) / temp
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    if c["op"] == "cross_entropy":
        loss = lse - (1.0 - c["smoothing"]) * x.gather(-1, t)
        if c["smoothing"]:
            loss = loss - c["smoothing"] * x.mean(-1, keepdim=True)
    else:
        loss = temp * temp * (p * (ln_p - x.gather(-1, t) + lse)).sum(-1, keepdim=True)
    back = lambda y: torch.where(live, y, 0.0).reshape(B, T)  # noqa: E731
    if c["direction"] == "forward":
        return back(loss), back(lse)
    dx = e / total
    if c.get("smoothing"):
        dx = dx - c["smoothing"] / V
    dx = dx.scatter_add(-1, t, -p.to(dx.dtype))
    dx = dx * torch.where(live, s["grad"].reshape(-1, 1) * temp, 0.0)
    dh = torch.matmul(dx, s["weight"]).reshape(B, T, D)
    return back(loss), back(lse), dh, torch.matmul(dx.T, h)


def _plain_embedding(s):
    c = s["case"]
    ids = s["ids"].reshape(-1)
    there = (ids >= 0) & (ids < c["V"])
    at = torch.where(there, ids, 0)
    res = []
    if c["direction"] != "backward":
        out = torch.where(there[:, None], s["table"][at] * s["scale"], 0.0)
        res.append(out.reshape(c["B"], c["T"], c["D"]))
    if c["direction"] != "forward":
        g = torch.where(there[:, None], s["grad"].reshape(-1, c["D"]), 0.0).double() * s["scale"]
        total = torch.zeros((c["V"], c["D"]), device=DEVICE, dtype=torch.float64).index_put((at,), g, accumulate=True)
        if c["accumulate"]:
            total = total + s["before"]
        res.append(total.to(s["grad"].dtype))
    return tuple(res)


# ---- the floor ----------------------------------------------------------------


def work(case):
    c = case
    N, V, D = c["B"] * c["T"], c["V"], c["D"]
    if c["op"] == "embedding":
        es = 8 if c["dtype"] == "f64" else 4
        # distinct tokens: the r-th comes up at least once in N with the share 1 / (r ln V)
        seen = min(V, int(N * (1 - c["padding"])), max(1, int(N / math.log(V) * (1 + math.log(max(1.0, V * math.log(V) / N))))))
        rows, b = N * (1 - c["padding"]), 0
        if c["direction"] != "backward":
            b += 8 * N + es * D * (seen + N)
        if c["direction"] != "forward":
            b += 8 * N + es * D * (rows + (2 * seen if c["accumulate"] else V))
            if c["accumulate"]:
                b += 2 * es * V * D  # the copy of the gradient that is there, which the pass makes
        return {"bytes": int(b), "flops": int(rows * D)}
    live = N * (1 - c["masked"])
    extra = 8 * N + 8 * N + (12 * N * c["K"] if c["op"] == "distillation" else 0)
    if c["direction"] == "forward":
        return {"bytes": int(4 * (live * D + V * D) + extra), "flops": int(2 * live * V * D)}
    return {"bytes": int(4 * (live * D + N * D + 2 * V * D) + 2 * extra), "flops": int(6 * live * V * D)}


# ---- the definition in 64 bits ---------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    V, D = c["V"], c["D"]
    if c["op"] == "embedding":
        ids = s["ids"].flatten()
        rows = ((ids >= 0) & (ids < V)).nonzero().flatten()
        res = []
        if c["direction"] != "backward":
            out = torch.zeros((ids.numel(), D), device=DEVICE, dtype=torch.float64)
            out[rows] = s["table"].double().index_select(0, ids[rows]).mul(s["scale"])
            res.append(out.view(c["B"], c["T"], D))
        if c["direction"] != "forward":
            gt = torch.zeros((V, D), device=DEVICE, dtype=torch.float64)
            order = torch.argsort(ids[rows], stable=True)
            gt.index_add_(0, ids[rows][order], s["grad"].double().flatten(0, 1)[rows][order], alpha=s["scale"])
            if c["accumulate"]:
                gt += s["before"].double()
            res.append(gt)
        return tuple(res)
    N = c["B"] * c["T"]
    loss = torch.zeros(N, device=DEVICE, dtype=torch.float64)
    lse = torch.zeros_like(loss)
    dh = torch.zeros((N, D), device=DEVICE, dtype=torch.float64)
    w = s["weight"].double().requires_grad_()
    dw = torch.zeros_like(w, requires_grad=False)
    temp = c.get("temperature", 1.0)
    ids = s["targets"].flatten()[:, None] if c["op"] == "cross_entropy" else s["ids"].flatten(0, 1)
    inside = (ids >= 0) & (ids < V)
    for rows in inside.any(-1).nonzero().flatten().split(max(1, (1 << 28) // V)):
        k = inside[rows]
        target = torch.zeros((len(rows), V), device=DEVICE, dtype=torch.float64)
        ln_p = torch.zeros((len(rows), 1), device=DEVICE, dtype=torch.float64)
        if c["op"] == "cross_entropy":
            target += c["smoothing"] / V
            target[torch.arange(len(rows), device=DEVICE), ids[rows, 0]] += 1.0 - c["smoothing"]
            entropy = ln_p[:, 0]
        else:
            z = s["logits"].flatten(0, 1)[rows].double().div(temp).masked_fill(~k, -math.inf)
            ln_p = torch.log_softmax(z, -1)
            p = ln_p.exp()
            target.scatter_add_(1, ids[rows].clamp(0, V - 1), p)
            entropy = (p * ln_p.masked_fill(~k, 0.0)).sum(-1)
        h = s["hidden"].flatten(0, 1)[rows].double().requires_grad_()
        x = h @ w.T / temp
        y = (temp * temp) * (entropy - (target * torch.log_softmax(x, -1)).sum(-1))
        loss[rows] = y.detach()
        lse[rows] = torch.logsumexp(x.detach(), -1)
        if c["direction"] == "train":
            a, b = torch.autograd.grad(y, (h, w), s["grad"].flatten()[rows].double())
            dh[rows] = a
            dw += b
        del x, y, target
    shape = (c["B"], c["T"])
    if c["direction"] == "forward":
        return loss.view(shape), lse.view(shape)
    return loss.view(shape), lse.view(shape), dh.view(*shape, D), dw
