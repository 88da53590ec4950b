"""fp32 calls of the cross entropy whose values span many powers of two: columns of unlike
units, a row far from the others, uneven weights, improbable entries.  The bounds are
elementwise, of the products that make an element up, with no share of the largest value of
a matrix.

An fp32 operand is three bf16 words (2^-27 left, products of words below 2^-26 left out):
2^-24 of each product.  A K-block of 64 is 4 steps of the largest words upon small ones, in
an accumulator that cuts 2^-22 of the sum a step and is then added at 2^-24."""

import pytest
import torch

import flash_vocab as F
import vocab_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
PROD = 2.0 ** -24


def chain(K):
    return 2.0 ** -22 * (1.125 * K / 16 + 8)


def bounds(X, W, t, bias, w, z):
    """loss, logZ and gradients in 64 bits, each with its elementwise bound."""
    X, W, w, z = (x.detach().double() for x in (X, W, w, z))
    (N, D), V = X.shape, W.shape[0]
    rows = torch.arange(N, device=DEV)
    c = torch.zeros(V, device=DEV, dtype=torch.float64) if bias is None else bias.detach().double()
    P, absS = X @ W.t(), X.abs() @ W.abs().t()
    S = P + c
    eS = (chain(D) + PROD) * absS + 2.0 ** -24 * S.abs()
    logZ = torch.logsumexp(S, 1)
    p = torch.exp(S - logZ[:, None])
    # logits off by eS move logZ by at most log sum p e^eS; then exp2 and log2 at 2^-21 of
    # arguments rounded at 2^-24 of up to 2^7, and a sum of at most V/32 + 64 roundings
    grow = torch.expm1(eS.clamp(max=60.0))
    ez = torch.log1p((p * grow).sum(1)) + 2.0 ** -17 + 2.0 ** -24 * (V / 32 + 64) \
        + 2.0 ** -22 * logZ.abs()
    at, e_at = S[rows, t], eS[rows, t]
    out = dict(loss=(logZ - at, ez + e_at + 2.0 ** -23 * at.abs()), logZ=(logZ, ez))
    a = w + z
    G = a[:, None] * p
    G[rows, t] -= w
    # p is at most 1; the stored g is rounded at 2^-27 and an exponential below 2^-126 is zero
    ep = torch.minimum(p * torch.expm1((eS + ez[:, None] + 2.0 ** -20).clamp(max=60.0)),
                       torch.ones_like(p))
    eG0 = a.abs()[:, None] * (ep + 2.0 ** -125) + 2.0 ** -24 * G.abs()
    eG = eG0 + 2.0 ** -26 * G.abs()
    out["dX"] = (G @ W, (eG @ W.abs() + (chain(V) + PROD) * (G.abs() @ W.abs())) * (1 + 2.0 ** -20))
    out["dW"] = (G.t() @ X, (eG.t() @ X.abs() + (chain(N) + PROD) * (G.abs().t() @ X.abs()))
                 * (1 + 2.0 ** -20))
    out["dbias"] = (G.sum(0), eG0.sum(0) + 2.0 ** -24 * (N / 32 + 64) * G.abs().sum(0))
    return out


def check(X, W, t, bias=None, w=None, z=None, skip=()):
    """Every row, except that rows `skip` have no usable bound of their own."""
    N = len(t)
    w = torch.ones(N, device=DEV) if w is None else w
    z = torch.zeros(N, device=DEV) if z is None else z
    leaves = [None if x is None else x.detach().clone().requires_grad_() for x in (X, W, bias)]
    loss, logZ = F.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction="none",
                                        return_logZ=True)
    ((loss * w).sum() + (logZ * z).sum()).backward()
    ref = bounds(X, W, t, bias, w, z)
    keep = torch.ones(N, dtype=torch.bool, device=DEV)
    for n in skip:
        keep[n] = False
    for got, name in ((loss.detach(), "loss"), (logZ.detach(), "logZ"), (leaves[0].grad, "dX")):
        R.assert_within(got[keep], ref[name][0][keep], ref[name][1][keep], name)
    R.assert_within(leaves[1].grad, *ref["dW"], "dW")
    if bias is not None:
        R.assert_within(leaves[2].grad, *ref["dbias"], "dbias")
    return ref


SIZES = pytest.mark.parametrize("N,V,D", [(17, 300, 32), (64, 300, 32), (700, 2100, 200)])


@SIZES
@pytest.mark.parametrize("power", [0, 8, 10])
def test_columns_of_unlike_units(N, V, D, power):
    X, W, t, c = R.problem(N, V, D, torch.float32, seed=N + power, bias=True)
    X[:, 3] *= 10.0 ** power
    W[:, 3] /= 10.0 ** power
    X[:, 7] /= 10.0 ** power
    W[:, 7] *= 10.0 ** power
    ref = check(X, W, t, c)
    assert float(ref["loss"][1].max()) < 1e-3      # the bound means something


@SIZES
@pytest.mark.parametrize("power", [9, 12])
def test_one_row_far_from_the_others(N, V, D, power):
    X, W, t, _ = R.problem(N, V, D, torch.float32, seed=N)
    X[5] *= 10.0 ** power
    ref = check(X, W, t, skip=[5])
    others = torch.arange(N, device=DEV) != 5
    assert float(ref["loss"][1][others].max()) < 1e-3


@SIZES
def test_one_entry_far_from_the_others(N, V, D):
    """Rows whose logit of that entry is very low see the other entries alone."""
    X, W, t, _ = R.problem(N, V, D, torch.float32, seed=N)
    t[t == 11] = 12
    W[11] *= 1e9
    S = X.double() @ W.double().t()
    X[S[:, 11] > 0] *= -1.0
    ref = check(X, W, t)
    assert float(ref["loss"][1].max()) < 1e-3


@SIZES
@pytest.mark.parametrize("span", [30, 60])
def test_weights_far_apart(N, V, D, span):
    """Each row of dX against its own weight, from 2^-span to 1."""
    X, W, t, c = R.problem(N, V, D, torch.float32, seed=3, bias=True)
    w = torch.exp2(-span * torch.rand(N, device=DEV))
    w[0], w[1] = 1.0, 2.0 ** -span
    z = 0.25 * w.flip(0)
    ref = check(X, W, t, c, w=w, z=z)
    # the bound means something beside the row's own weights
    relative = ref["dX"][1].amax(1) / ((w + z) * W.abs().max())
    assert float(relative.max()) < 1e-3


@SIZES
def test_improbable_entries(N, V, D):
    """Rows of dW whose probabilities are 1e-13 to 1e-20 in every row of X."""
    X, W, t, c = R.problem(N, V, D, torch.float32, seed=8, bias=True)
    rare = torch.zeros(V, dtype=torch.bool, device=DEV)
    rare[::3] = True
    t[rare[t]] = 1
    c[rare] -= torch.linspace(30, 45, int(rare.sum()), device=DEV)
    ref = check(X, W, t, c)
    value, bound = ref["dW"]
    assert float((bound[rare].max(1).values / value[rare].abs().max(1).values).max()) < 1e-3


def test_the_ends_of_the_range():
    """Values near the largest float against values near the smallest normal ones."""
    X, W, t, _ = R.problem(40, 90, 24, torch.float32, seed=2)
    X[:, 0] = 3.4e38 * torch.sign(X[:, 0])
    W[:, 0] *= 2.0 ** -127
    X[:, 1] *= 2.0 ** -100
    W[:, 1] *= 2.0 ** 90
    ref = bounds(X, W, t, None, torch.ones(40, device=DEV), torch.zeros(40, device=DEV))
    loss, logZ = F.linear_cross_entropy(X, W, t, reduction="none", return_logZ=True)
    # words of values below 2^-110 fall out of bf16's normal range: 2^-133 of 3.4e38, 2^-5
    # ... of a weight's last word at most, so the logits carry 2^-133 x 2^128 a word
    off = 3 * 2.0 ** -5
    R.assert_within(loss, ref["loss"][0], ref["loss"][1] + 2 * off, "loss")
    R.assert_within(logZ, ref["logZ"][0], ref["logZ"][1] + off, "logZ")


def test_many_pieces_of_rows_and_entries():
    """Several chunks of rows and pieces of the vocabulary, weights and columns uneven."""
    N, V, D = 3000, 9001, 70
    X, W, t, c = R.problem(N, V, D, torch.float32, seed=6, bias=True)
    X[:, 2] *= 1e7
    W[:, 2] /= 1e7
    w = torch.exp2(-25 * torch.rand(N, device=DEV))
    check(X, W, t, c, w=w)
