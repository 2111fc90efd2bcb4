"""Cases, inputs and plain forms of the training operators around the expert
layers: the vocabulary's linear cross entropy, the token embedding and the
routing balance loss, each with its gradients."""

import math

import torch

own = False

IGNORE = -100


def listed():
    return [
        # --- linear cross entropy: hidden [T, d] against the output table [V, d]
        # log-likelihood of the one next token of a request (latency of one read of the table)
        dict(name="ce_eval_1", op="ce", T=1, V=100277, d=1024, dtype="bf16", train=False, reduction="none", ignored=0.0),
        # per-token log-likelihoods of an odd number of held-out tokens
        dict(name="ce_eval_4095", op="ce", T=4095, V=100277, d=1024, dtype="bf16", train=False, reduction="none",
             ignored=0.0),
        # fine-tuning on one short answer: most of the prompt's labels are ignored
        dict(name="ce_train_300", op="ce", T=300, V=100277, d=1024, dtype="bf16", train=True, reduction="mean",
             ignored=0.6),
        # a pre-training step of the whole decoder: 8 sequences of 2048, the last label of each ignored
        dict(name="ce_train_16384", op="ce", T=16384, V=100277, d=1024, dtype="bf16", train=True, reduction="mean",
             ignored=1.0 / 2048),
        # an fp32 model with a small odd vocabulary, per-token losses weighted by the caller
        dict(name="ce_train_f32", op="ce", T=2047, V=32003, d=512, dtype="f32", train=True, reduction="none",
             ignored=0.1),
        # --- embedding: the tied table's other end
        # the tokens of a small decoding batch
        dict(name="emb_lookup_8", op="emb", T=8, V=100277, d=1024, dtype="bf16", train=False, scale=1.0, padding=-1),
        # the same pre-training step: lookup and the table's gradient, Zipf-distributed tokens
        dict(name="emb_train_16384", op="emb", T=16384, V=100277, d=1024, dtype="bf16", train=True, scale=1.0,
             padding=-1),
        # fp32 with the sqrt(d) scale, an odd width, and a padding token that a fifth of the batch holds
        dict(name="emb_train_f32", op="emb", T=4099, V=32003, d=515, dtype="f32", train=True, scale=515 ** 0.5,
             padding=0),
        # --- balance loss over the router's choices
        # a small layer's short batch
        dict(name="bal_256", op="bal", T=256, H=8, k=16, N=4096, dtype="f32", ids="i32", masked=0.0),
        # one layer of the pre-training step
        dict(name="bal_16384", op="bal", T=16384, H=8, k=16, N=262144, dtype="f32", ids="i32", masked=1.0 / 16),
        # weights and ids as the router module hands them out, a long batch
        dict(name="bal_65536_bf16", op="bal", T=65536, H=8, k=16, N=262144, dtype="bf16", ids="i64", masked=0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ce", "ce", "emb", "bal"])
    if op == "ce":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        T = _log_int(rng, 1, 16384 if dtype == "bf16" else 4096)
        V = _log_int(rng, 1000, 131072 if dtype == "bf16" else 65536)
        d = _log_int(rng, 64, 2048)
        if rng.random() < 0.7:
            d = max(64, d // 8 * 8)
        # no dearer than the largest listed case, in products and in logits
        T = max(1, min(T, 16384 * 100277 * 1024 // (V * d), 16384 * 100277 // V))
        train = rng.random() < 0.7
        return dict(op="ce", T=T, V=V, d=d, dtype=dtype, train=train,
                    reduction=rng.choice(["mean", "mean", "sum", "none"]), ignored=rng.choice([0.0, 0.05, 0.6]))
    if op == "emb":
        V = _log_int(rng, 1000, 131072)
        return dict(op="emb", T=_log_int(rng, 1, 65536), V=V, d=_log_int(rng, 64, 2048),
                    dtype=rng.choice(["bf16", "f32"]), train=rng.random() < 0.7,
                    scale=rng.choice([1.0, 0.5, 22.627]), padding=rng.choice([-1, 0, V - 1]))
    side = rng.randint(32, 512)
    return dict(op="bal", T=_log_int(rng, 1, 65536), H=rng.choice([1, 2, 4, 8]), k=rng.choice([4, 8, 16]),
                N=side * side, dtype=rng.choice(["f32", "bf16"]), ids=rng.choice(["i32", "i64"]),
                masked=rng.choice([0.0, 0.1, 0.5]))


_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _zipf(n, V, g):
    """Token ids with frequencies 1 / rank^1.1; frequent tokens have low ids,
    as in a byte-pair vocabulary."""
    w = torch.arange(1, V + 1, device="cuda", dtype=torch.float64).pow(-1.1)
    c = torch.cumsum(w / w.sum(), 0)
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    return torch.searchsorted(c, u).clamp_(max=V - 1)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["op"] == "ce":
        T, V, d, dt = case["T"], case["V"], case["d"], _DT[case["dtype"]]
        W = torch.randn(V, d, generator=g, device="cuda") * d ** -0.5
        y = _zipf(T, V, g)
        # normalised states that know their label more or less well: from a
        # flat distribution to nearly all of the probability on one token
        h = torch.randn(T, d, generator=g, device="cuda")
        h += W[y] * torch.rand(T, 1, generator=g, device="cuda") * 16.0
        y[torch.rand(T, generator=g, device="cuda") < case["ignored"]] = IGNORE
        y[0] = 0
        s["h"] = h.to(dt)
        s["W"] = W.to(dt)
        s["y"] = y
        s["g"] = None
        if case["reduction"] == "none":
            s["g"] = torch.rand(T, generator=g, device="cuda") + 0.5
        if case["train"]:
            s["h"].requires_grad_(True)
            s["W"].requires_grad_(True)
    elif case["op"] == "emb":
        T, V, d, dt = case["T"], case["V"], case["d"], _DT[case["dtype"]]
        s["W"] = (torch.randn(V, d, generator=g, device="cuda") * 0.02).to(dt)
        ids = _zipf(T, V, g)
        pad = case["padding"]
        if pad >= 0:
            ids[torch.rand(T, generator=g, device="cuda") < 0.2] = pad
        s["ids"] = ids
        s["pad"] = pad if pad >= 0 else None
        if case["train"]:
            s["dy"] = (torch.randn(T, d, generator=g, device="cuda") * 1e-3).to(dt)
            s["W"].requires_grad_(True)
    else:
        T, H, k, N = case["T"], case["H"], case["k"], case["N"]
        # popular and unpopular experts: the router's choices crowd the low ids
        u = torch.rand(T, H, k, generator=g, device="cuda", dtype=torch.float64)
        s["ids"] = (u.pow(2.0) * N).long().clamp_(max=N - 1).to(torch.int32 if case["ids"] == "i32" else torch.int64)
        w = torch.softmax(torch.randn(T, H, k, generator=g, device="cuda"), -1).to(_DT[case["dtype"]])
        s["w"] = w.requires_grad_(True)
        s["mask"] = None
        if case["masked"] > 0:
            m = torch.rand(T, generator=g, device="cuda") >= case["masked"]
            m[0] = True
            s["mask"] = m
        s["g"] = torch.full((), 0.01, device="cuda")
    return s


# ------------------------------------------------------------ plain forms --
def _plain_ce(s):
    h, W, y = s["h"].detach(), s["W"].detach(), s["y"]
    h32, W32 = h.float(), W.float()
    valid = y != IGNORE
    at = torch.where(valid, y, torch.zeros_like(y))
    logits = h32 @ W32.t()
    top = logits.amax(1, keepdim=True)
    label = logits.gather(1, at[:, None])[:, 0]
    e = logits.sub_(top).exp_()
    total = e.sum(1, keepdim=True)
    loss = torch.where(valid, total.log()[:, 0] + top[:, 0] - label, 0.0)
    n = valid.sum()
    if s["reduction"] == "none":
        out = loss
    elif s["reduction"] == "sum":
        out = loss.sum()
    else:
        out = loss.sum() / n
    if not s["train"]:
        return [out]
    if s["reduction"] == "none":
        g = s["g"]
    elif s["reduction"] == "sum":
        g = torch.ones_like(loss)
    else:
        g = torch.ones_like(loss) / n
    g = torch.where(valid, g, 0.0)
    p = e.div_(total)
    rows = torch.arange(y.shape[0], device=y.device)
    p[rows, at] -= 1.0
    dl = p.mul_(g[:, None])
    return [out, (dl @ W32).to(h.dtype), (dl.t() @ h32).to(W.dtype)]


def _plain_emb(s):
    W, ids = s["W"].detach(), s["ids"]
    out = (W[ids].float() * s["scale"]).to(W.dtype)
    if not s["train"]:
        return [out]
    dy = s["dy"].float() * s["scale"]
    dW = torch.zeros(W.shape, dtype=torch.float32, device=W.device)
    dW.index_add_(0, ids, dy)
    if s["pad"] is not None:
        dW[s["pad"]] = 0.0
    return [out, dW.to(W.dtype)]


def _plain_bal(s):
    w, ids, N = s["w"].detach().float(), s["ids"].long(), s["N"]
    T, H, k = w.shape
    m = s["mask"] if s["mask"] is not None else torch.ones(T, dtype=torch.bool, device=w.device)
    one = m.to(torch.int32)[:, None, None].expand(T, H, k)
    counts = torch.zeros(N, dtype=torch.int32, device=w.device)
    counts.index_add_(0, ids.reshape(-1), one.reshape(-1))
    n = m.sum().float().clamp(min=1.0)
    coef = N / (n * n * (H * H * k))
    per = counts[ids].float() * m[:, None, None] * coef
    loss = (w * per).sum()
    return [loss, counts, (per * s["g"]).to(s["w"].dtype)]


# ------------------------------------------------------------ one pass --
def run(s):
    if not own:
        with torch.no_grad():
            return {"ce": _plain_ce, "emb": _plain_emb, "bal": _plain_bal}[s["op"]](s)
    from ethos_b200 import functional as EF
    if s["op"] == "ce":
        if not s["train"]:
            with torch.no_grad():
                return [EF.linear_cross_entropy(s["h"], s["W"], s["y"], ignore_index=IGNORE,
                                                reduction=s["reduction"])]
        loss = EF.linear_cross_entropy(s["h"], s["W"], s["y"], ignore_index=IGNORE, reduction=s["reduction"])
        dh, dW = torch.autograd.grad(loss, (s["h"], s["W"]), s["g"])
        return [loss.detach(), dh, dW]
    if s["op"] == "emb":
        if not s["train"]:
            with torch.no_grad():
                return [EF.embedding(s["ids"], s["W"], scale=s["scale"], padding_idx=s["pad"])]
        out = EF.embedding(s["ids"], s["W"], scale=s["scale"], padding_idx=s["pad"])
        dW, = torch.autograd.grad(out, s["W"], s["dy"])
        return [out.detach(), dW]
    loss, counts = EF.balance_loss(s["w"], s["ids"], s["N"], mask=s["mask"])
    dw, = torch.autograd.grad(loss, s["w"], s["g"])
    return [loss.detach(), counts, dw]


def work(case):
    if case["op"] == "ce":
        T, V, d = case["T"], case["V"], case["d"]
        e = 2 if case["dtype"] == "bf16" else 4
        # ignored rows need no products
        live = max(1.0, T * (1.0 - case["ignored"]))
        io = (T * d + V * d) * e + 8 * T + (4 * T if case["reduction"] == "none" else 4)
        if case["train"]:
            return {"bytes": io + (T * d + V * d) * e, "flops": 6.0 * live * V * d}
        return {"bytes": io, "flops": 2.0 * live * V * d}
    if case["op"] == "emb":
        T, V, d = case["T"], case["V"], case["d"]
        e = 2 if case["dtype"] == "bf16" else 4
        b = 8 * T + 2 * T * d * e
        if case["train"]:
            return {"bytes": b + (T * d + V * d) * e, "flops": 2.0 * T * d}
        return {"bytes": b, "flops": 1.0 * T * d}
    n = case["T"] * case["H"] * case["k"]
    e = 2 if case["dtype"] == "bf16" else 4
    i = 4 if case["ids"] == "i32" else 8
    return {"bytes": n * (i + 2 * e) + 4 * case["N"] + (case["T"] if case["masked"] > 0 else 0), "flops": 3.0 * n}


# ------------------------------------------------------------ 64 bits --
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "ce":
            return _exact_ce(case, s)
        if case["op"] == "emb":
            W = s["W"].detach().double()
            out = torch.index_select(W, 0, s["ids"]) * case["scale"]
            if not case["train"]:
                return [out]
            ids, dy = s["ids"], s["dy"].double()
            if s["pad"] is not None:
                dy = dy * (ids != s["pad"]).double()[:, None]
            order = torch.argsort(ids, stable=True)
            total = torch.cat([torch.zeros(1, dy.shape[1], dtype=torch.float64, device=dy.device),
                               torch.cumsum(dy[order], 0)])
            edges = torch.searchsorted(ids[order], torch.arange(case["V"] + 1, device=ids.device))
            return [out, (total[edges[1:]] - total[edges[:-1]]) * case["scale"]]
        T, H, k, N = case["T"], case["H"], case["k"], case["N"]
        w, ids = s["w"].detach().double(), s["ids"].long()
        m = torch.ones(T, device="cuda", dtype=torch.float64) if s["mask"] is None else s["mask"].double()
        flat = ids.reshape(-1)
        live = m[:, None, None].expand(T, H, k).reshape(-1)
        counts = torch.bincount(flat, weights=live, minlength=N)
        mass = torch.bincount(flat, weights=live * w.reshape(-1), minlength=N)
        n = max(1.0, float(m.sum()))
        loss = N * ((counts / (n * H * k)) * (mass / (n * H))).sum()
        dw = (live * (counts / (n * H * k))[flat] * (N / (n * H))).reshape(T, H, k) * float(s["g"])
        return [loss, counts.to(torch.int32), dw]


def _exact_ce(case, s):
    h, W, y = s["h"].detach(), s["W"].detach().double(), s["y"]
    T, V, d = case["T"], case["V"], case["d"]
    valid = y != IGNORE
    n = float(valid.sum())
    loss = torch.zeros(T, dtype=torch.float64, device="cuda")
    dh = torch.zeros(T, d, dtype=torch.float64, device="cuda") if case["train"] else None
    dW = torch.zeros(V, d, dtype=torch.float64, device="cuda") if case["train"] else None
    step = max(1, min(T, (1 << 28) // V))
    for a in range(0, T, step):
        hb, yb, vb = h[a:a + step].double(), y[a:a + step], valid[a:a + step]
        logp = torch.log_softmax(hb @ W.t(), dim=1)
        pick = torch.nn.functional.one_hot(torch.where(vb, yb, 0), V) if V * hb.shape[0] <= 1 << 24 else None
        got = logp.gather(1, torch.where(vb, yb, 0)[:, None])[:, 0]
        loss[a:a + step] = torch.where(vb, -got, 0.0)
        if not case["train"]:
            continue
        scale = {"none": s["g"][a:a + step].double() if s["g"] is not None else None, "sum": torch.ones_like(got),
                 "mean": torch.full_like(got, 1.0 / n)}[case["reduction"]]
        scale = torch.where(vb, scale, 0.0)
        p = logp.exp_()
        if pick is not None:
            p = p - pick
        else:
            p.scatter_add_(1, torch.where(vb, yb, 0)[:, None], torch.full_like(got, -1.0)[:, None])
        p = p * scale[:, None]
        dh[a:a + step] = p @ W
        dW += p.t() @ hb
    out = {"none": loss, "sum": loss.sum(), "mean": loss.sum() / n}[case["reduction"]]
    return [out, dh, dW] if case["train"] else [out]
