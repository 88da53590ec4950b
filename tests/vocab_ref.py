"""Plain 64-bit forms of the vocabulary operators and the error bounds their
kernels are held to (elementwise, from the arithmetic; no fitted constants).

u is half a step of the element type (2^-8 bf16, 2^-11 fp16, 2^-24 fp32).  fp32
operands run as three bf16 words each, which carry a relative error of 2^-24 per
product together (held to 2^-21 here); bf16 and fp16 products are exact in fp32.

An fp32 sum of K products on the tensor core is kept in steps of 16, each
cutting the running sum at 2^-23 of its magnitude and the aligned products at
another 2^-23 of the largest: at most 2^-22 (K/16 + 8) sum|a||b|, 8 for the
joining of parts.
"""

import torch

IGNORE = -100
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
PROD = {torch.bfloat16: 0.0, torch.float16: 0.0, torch.float32: 2.0 ** -21}
# half a step at the small end; fp32 and bf16 values below 2^-126 may be flushed to zero
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}


def chain(K):
    return 2.0 ** -22 * (K / 16 + 8)


def xent(X, W, t, bias, ignore=IGNORE, w=None, dlogZ=None):
    """dict with loss, logZ, their bound, and for weights w (N,) of the losses
    (and dlogZ) the gradients with their bounds.  Everything in float64."""
    kind = X.dtype
    X, W = X.detach().double(), W.detach().double()
    V, D = W.shape
    keep = t != ignore
    X = torch.where(keep[:, None], X, torch.zeros_like(X))
    P = X @ W.t()
    absS = X.abs() @ W.abs().t()
    c = torch.zeros(V, dtype=torch.float64, device=X.device) if bias is None \
        else bias.detach().double()
    S = P + c
    logZ = torch.logsumexp(S, 1)
    rows = torch.arange(len(t), device=X.device)
    at = S[rows, t.clamp(0, V - 1)]
    finite_c = torch.where(torch.isinf(c), torch.zeros_like(c), c)
    # logit error: the product sum, and one rounding with the bias
    eS = (chain(D) + PROD[kind]) * absS.amax(1) + 2.0 ** -24 * (P + finite_c).abs().amax(1)
    # exp2/log2 at 2^-21 relative (arguments rounded at 2^-24 of up to 2^7), sums of V
    # positive terms kept in at most V/32 + 64 roundings of 2^-24
    ez = eS + 2.0 ** -17 + 2.0 ** -24 * (V / 32 + 64) + 2.0 ** -22 * logZ.abs()
    out = dict(loss=torch.where(keep, logZ - at, torch.zeros_like(at)),
               logZ=torch.where(keep, logZ, torch.zeros_like(at)),
               e_loss=ez + eS + 2.0 ** -23 * at.abs(), e_logZ=ez)
    if w is None:
        return out
    b = torch.where(keep, w.double(), torch.zeros_like(at))
    a = b if dlogZ is None else b + torch.where(keep, dlogZ.double(), torch.zeros_like(at))
    p = torch.where(keep[:, None], torch.exp(S - logZ[:, None]), torch.zeros_like(S))
    G = a[:, None] * p
    G[rows, t.clamp(0, V - 1)] -= b
    # g is stored in the element type (fp32: two fp16 words, 2^-21); fp16 words hold
    # g scaled to a maximum of at least 2^11, with steps of 2^-24 at the small end
    ug = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -21}[kind]
    top = max(float(a.abs().max()), float(b.abs().max())) if len(t) else 0.0
    # and an fp32 exponential below 2^-126 is zero: at most that times a is lost
    small = 2.0 ** -125 * max(top, 1.0) if kind == torch.bfloat16 else 2.0 ** -35 * top
    eG = G.abs() * ug + (a.abs() * (2 * ez + 2.0 ** -20))[:, None] * p + small * keep[:, None]
    out["dX"], out["dW"], out["dbias"] = G @ W, G.t() @ X, G.sum(0)
    u, tiny = U[kind], TINY[kind]
    eG0 = eG - G.abs() * ug                       # dbias is summed before g is rounded
    out["e_dX"] = (eG @ W.abs() + (chain(V) + PROD[kind]) * (G.abs() @ W.abs())) * (1 + u) \
        + u * out["dX"].abs() + tiny
    out["e_dW"] = (eG.t() @ X.abs() + (chain(len(t)) + PROD[kind]) * (G.abs().t() @ X.abs())) \
        * (1 + u) + u * out["dW"].abs() + tiny
    out["e_dbias"] = eG0.sum(0) + 2.0 ** -24 * (len(t) / 32 + 64) * G.abs().sum(0)
    return out


def assert_within(got, ref, bound, what):
    got = got.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    nan = torch.isnan(ref) | torch.isinf(ref)
    same = (torch.isnan(got) & torch.isnan(ref)) | (got == ref)
    err = (got - ref).abs()
    ok = torch.where(nan, same, err <= bound)
    if not bool(ok.all()):
        bad = (~ok).nonzero()[0].tolist()
        b = bound.expand_as(ref) if torch.is_tensor(bound) else torch.full_like(ref, bound)
        raise AssertionError(f"{what}: {int((~ok).sum())} of {ok.numel()} out of bound, first at "
                             f"{bad}: {float(got[tuple(bad)])} vs {float(ref[tuple(bad)])}, "
                             f"bound {float(b[tuple(bad)])}")


def embed_grad(g, ids, V, scale, ignore=IGNORE):
    """(dtable, bound): sums of n rows keep at most n roundings of 2^-24 each way."""
    u, tiny = U[g.dtype], TINY[g.dtype]
    live = (ids != ignore) & (ids >= 0) & (ids < V)
    G = g.double()[live]
    d = torch.zeros(V, g.shape[1], dtype=torch.float64, device=g.device)
    mag = torch.zeros_like(d)
    d.index_add_(0, ids[live], G)
    mag.index_add_(0, ids[live], G.abs())
    n = torch.bincount(ids[live], minlength=V).double()[:, None]
    d, mag = d * scale, mag * abs(scale)
    return d, (2.0 ** -24 * (n + 3)) * mag * (1 + u) + u * d.abs() + tiny


def problem(N, V, D, dtype, seed=0, ignored=0.0, bias=False, device="cuda", spread=2.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    W = torch.randn(V, D, generator=g) * (spread / D ** 0.5)
    t = torch.randint(0, V, (N,), generator=g)
    X = torch.randn(N, D, generator=g) + 1.5 * torch.rand(N, 1, generator=g) * W[t]
    if ignored:
        t[torch.rand(N, generator=g) < ignored] = IGNORE
    c = torch.log_softmax(torch.randn(V, generator=g), 0) if bias else None
    return (X.to(dtype).to(device), W.to(dtype).to(device), t.to(device),
            None if c is None else c.to(device))
