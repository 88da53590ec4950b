"""Cases of the vocabulary operators: the linear cross entropy with its gradient
and the scaled embedding lookup with its gradient.

``run`` computes a case in its plain form (torch operations in 32 bits) or,
where ``own`` is set, through ``flash_vocab``."""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

IGNORE = -100
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _flash_vocab():
    if "flash_vocab" not in sys.modules:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                           "flash-gmm_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
    import flash_vocab
    return flash_vocab


def listed():
    return [
        # the score of one generated token: bound by reading the table, and by latency
        dict(name="score one token", op="score", type="bf16", N=1, V=32768, D=1024,
             ignored=0.0, bias=False),
        # the scores of a short answer, with odd sizes that no tile divides
        dict(name="score an answer, odd", op="score", type="fp16", N=37, V=50021, D=1003,
             ignored=0.0, bias=True),
        # an evaluation batch: the loss alone
        dict(name="evaluation batch", op="score", type="bf16", N=4096, V=32768, D=2048,
             ignored=0.0, bias=False),
        # a training step's loss and gradients, a tenth of the positions padded
        dict(name="training batch", op="train", type="bf16", N=8192, V=65536, D=2048,
             ignored=0.1, bias=False),
        # the same with odd sizes and a bias, over a small vocabulary
        dict(name="training batch, odd", op="train", type="fp16", N=1021, V=10007, D=777,
             ignored=0.05, bias=True),
        # a small model trained in full precision
        dict(name="training batch, fp32", op="train", type="fp32", N=2048, V=16384, D=512,
             ignored=0.0, bias=False),
        # labelled rows against the components of the headline mixture (K=1024, D=128)
        dict(name="labelled mixture", op="train", type="fp32", N=131072, V=1024, D=128,
             ignored=0.0, bias=True),
        # the input row of one generated token
        dict(name="lookup of one token", op="lookup", type="bf16", N=1, V=32768, D=1024,
             ignored=0.0),
        # the input rows of a prompt batch
        dict(name="lookup of a batch", op="lookup", type="bf16", N=16384, V=65536, D=2048,
             ignored=0.0),
        # lookup and gradient of a training batch, padded positions among it
        dict(name="embedding step", op="embed", type="bf16", N=16384, V=65536, D=2048,
             ignored=0.1),
        # the same in full precision with odd sizes
        dict(name="embedding step, odd", op="embed", type="fp32", N=10007, V=5003, D=333,
             ignored=0.0),
    ]


def _spread(rng, lo, hi):
    """A whole number, spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["score", "score", "train", "train", "lookup", "embed"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("score", "train"):
        while True:
            N, V, D = (_spread(rng, 1, 65536), _spread(rng, 128, 131072), _spread(rng, 32, 4096))
            # no more work than the largest listed case of its type's kind
            if N * V * D <= (1.0e12 if kind != "fp32" else 1.5e11) and N * V <= 5.0e8:
                break
        if rng.random() < 0.5:  # half of the cases have the widths that models have
            D = max(32, D // 64 * 64)
        return dict(op=op, type=kind, N=N, V=V, D=D, ignored=rng.choice([0.0, 0.0, 0.1, 0.4]),
                    bias=rng.random() < 0.3)
    while True:
        N, V, D = (_spread(rng, 1, 65536), _spread(rng, 128, 131072), _spread(rng, 32, 4096))
        if V * D <= 1.3e8 and N * D <= 3.3e7:
            break
    if rng.random() < 0.5:
        D = max(32, D // 64 * 64)
    return dict(op=op, type=kind, N=N, V=V, D=D, ignored=rng.choice([0.0, 0.1]))


def _tokens(g, N, V, ignored):
    """Tokens with the long tail that text has (density ~ 1/v), scattered over the table."""
    u = torch.rand(N, generator=g, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(V + 1)) - 1).long().clamp_(0, V - 1)
    perm = torch.randperm(V, generator=g, device="cuda")
    t = perm[rank]
    if ignored > 0:   # the first position of a batch always holds a token
        t[1:][torch.rand(N - 1, generator=g, device="cuda") < ignored] = IGNORE
    return t


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    N, V, D, dt = case["N"], case["V"], case["D"], TYPES[case["type"]]
    s = dict(case)
    s["t"] = _tokens(g, N, V, case["ignored"])
    # rows of unit variance; logits of a deviation of about 2
    W = torch.randn(V, D, generator=g, device="cuda") * (2.0 / math.sqrt(D))
    if case["op"] in ("score", "train"):
        X = torch.randn(N, D, generator=g, device="cuda")
        # the model knows something: each row leans towards its token's vector
        X += W[s["t"].clamp_min(0)] * (1.5 * torch.rand(N, 1, generator=g, device="cuda"))
        train = case["op"] == "train"
        s["X"] = X.to(dt).requires_grad_(train)
        s["W"] = W.to(dt).requires_grad_(train)
        s["bias"] = None
        if case["bias"]:
            c = torch.log_softmax(torch.randn(V, generator=g, device="cuda"), 0)
            s["bias"] = c.requires_grad_(train)
    else:
        s["scale"] = math.sqrt(D)
        s["W"] = W.to(dt).requires_grad_(case["op"] == "embed")
        if case["op"] == "embed":
            s["g"] = torch.randn(N, D, generator=g, device="cuda").to(dt)
    return s


def _plain_score(s):
    X, W, t, bias = s["X"].detach().float(), s["W"].detach().float(), s["t"], s["bias"]
    S = X @ W.t()
    if bias is not None:
        S += bias.detach()
    keep = t != IGNORE
    m = S.max(1).values
    at = S.gather(1, t.clamp_min(0)[:, None])[:, 0]
    e = S.sub_(m[:, None]).exp_()
    z = e.sum(1)
    logZ = m + z.log()
    loss = logZ - at
    zero = torch.zeros_like(loss)
    return torch.where(keep, loss, zero), torch.where(keep, logZ, zero), keep, e, z


def _plain_train(s):
    loss, _, keep, e, z = _plain_score(s)
    X, W, t = s["X"].detach(), s["W"].detach(), s["t"]
    count = keep.double().sum()
    mean = (loss.double().sum() / count).float()
    w = keep / count.float()                      # each row's weight in the mean
    G = e.mul_((w / z)[:, None])
    G[torch.arange(len(t), device=t.device), t.clamp_min(0)] -= w
    out = dict(loss=mean, dX=(G @ W.float()).to(X.dtype), dW=(G.t() @ X.float()).to(W.dtype))
    if s["bias"] is not None:
        out["dbias"] = G.sum(0)
    return out


def _plain_lookup(s):
    W, t = s["W"].detach(), s["t"]
    rows = W[t.clamp_min(0)].float() * s["scale"]
    return torch.where((t != IGNORE)[:, None], rows, torch.zeros_like(rows)).to(W.dtype)


def _plain_embed(s):
    W, t, g = s["W"].detach(), s["t"], s["g"]
    keep = t != IGNORE
    d = torch.zeros(W.shape, device=W.device, dtype=torch.float32)
    d.index_add_(0, t[keep], g[keep].float())
    return dict(out=_plain_lookup(s), dW=(d * s["scale"]).to(W.dtype))


def run(state):
    s = state
    if not own:
        if s["op"] == "score":
            loss, logZ = _plain_score(s)[:2]
            return dict(loss=loss, logZ=logZ)
        return {"train": _plain_train, "lookup": _plain_lookup, "embed": _plain_embed}[s["op"]](s)
    F = _flash_vocab()
    if s["op"] == "score":
        loss, logZ = F.linear_cross_entropy(s["X"], s["W"], s["t"], s["bias"], reduction="none",
                                            return_logZ=True)
        return dict(loss=loss, logZ=logZ)
    if s["op"] == "train":
        loss = F.linear_cross_entropy(s["X"], s["W"], s["t"], s["bias"])
        leaves = (s["X"], s["W"]) if s["bias"] is None else (s["X"], s["W"], s["bias"])
        grads = torch.autograd.grad(loss, leaves)
        out = dict(loss=loss.detach(), dX=grads[0], dW=grads[1])
        if s["bias"] is not None:
            out["dbias"] = grads[2]
        return out
    rows = F.embedding_lookup(s["W"], s["t"], scale=s["scale"])
    if s["op"] == "lookup":
        return rows
    return dict(out=rows.detach(), dW=torch.autograd.grad(rows, s["W"], s["g"])[0])


def work(case):
    N, V, D, b = case["N"], case["V"], case["D"], SIZE[case["type"]]
    live = N * (1.0 - case["ignored"])
    if case["op"] == "score":
        return {"bytes": b * D * (live + V) + 8 * N + 8 * N + (4 * V if case["bias"] else 0),
                "flops": 2.0 * live * V * D}
    if case["op"] == "train":
        return {"bytes": b * D * (live + N + 2 * V) + 8 * N + (8 * V if case["bias"] else 0),
                "flops": 6.0 * live * V * D}
    # distinct rows of the table that tokens of density ~ 1/v reach
    rows = min(live, V * math.log1p(live / math.log(V + 1)) / math.log(V + 1))
    lookup = b * D * (rows + N) + 8 * N
    if case["op"] == "lookup":
        return {"bytes": lookup, "flops": live * D}
    return {"bytes": lookup + b * D * (live + V), "flops": 2.0 * live * D + V * D}


def exact(case, seed):
    s = prepare(case, seed)
    N, V, D, t = case["N"], case["V"], case["D"], s["t"]
    W = s["W"].detach().double()
    if case["op"] in ("lookup", "embed"):
        valid = (t >= 0).nonzero()[:, 0]
        out = torch.zeros(N, D, device="cuda", dtype=torch.float64)
        out[valid] = W[t[valid]] * s["scale"]
        if case["op"] == "lookup":
            return out
        order = t[valid].argsort(stable=True)
        ids, counts = t[valid][order].unique_consecutive(return_counts=True)
        ends = counts.cumsum(0)
        dW = torch.zeros(V, D, device="cuda", dtype=torch.float64)
        step = max(1, (1 << 25) // max(1, N))     # columns at a time: running sums, differences
        for d in range(0, D, step):
            run_sum = s["g"][valid, d:d + step].double()[order].cumsum(0)
            upto = run_sum[ends - 1]
            dW[ids, d:d + step] = torch.diff(upto, dim=0, prepend=torch.zeros_like(upto[:1]))
        return dict(out=out, dW=dW * s["scale"])
    X = s["X"].detach().double()
    c = torch.zeros(V, device="cuda", dtype=torch.float64)
    if s["bias"] is not None:
        c = s["bias"].detach().double()
    loss = torch.zeros(N, device="cuda", dtype=torch.float64)
    logZ = torch.zeros(N, device="cuda", dtype=torch.float64)
    train = case["op"] == "train"
    count = int((t >= 0).sum())
    if train:
        dX, dW, dc = torch.zeros_like(X), torch.zeros_like(W), torch.zeros_like(c)
    rows = max(1, (1 << 27) // V)
    for n in range(0, N, rows):
        part = (t[n:n + rows] >= 0).nonzero()[:, 0] + n
        if part.numel() == 0:
            continue
        logits = torch.addmm(c, X[part], W.t())
        lz = torch.logsumexp(logits, 1)
        logp = logits - lz[:, None]
        hot = torch.nn.functional.nll_loss(logp, t[part], reduction="none")
        loss[part], logZ[part] = hot, lz
        if train:
            G = logp.exp_()
            G.scatter_add_(1, t[part][:, None], -torch.ones_like(lz)[:, None])
            G /= count
            dX[part] = G @ W
            dW += G.t() @ X[part]
            dc += G.sum(0)
    if not train:
        return dict(loss=loss, logZ=logZ)
    out = dict(loss=loss.sum() / count, dX=dX, dW=dW)
    if s["bias"] is not None:
        out["dbias"] = dc
    return out
