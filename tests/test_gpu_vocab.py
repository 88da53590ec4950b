"""The vocabulary operators (flash_vocab) on the GPU against plain 64-bit forms,
within bounds derived from the arithmetic (vocab_ref)."""

import math

import pytest
import torch

import _fgmm_lib as L
import flash_gmm
import flash_vocab as F
import vocab_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FH, FS = torch.bfloat16, torch.float16, torch.float32


def check_xent(X, W, t, bias=None, *, reduction="none", wantgrad=True, seed=1, **kw):
    """Forward and all gradients of a weighted sum of loss and logZ."""
    N = t.numel()
    g = torch.Generator(device="cpu").manual_seed(seed)
    w = (torch.rand(N, generator=g) + 0.5).to(DEV)
    z = (0.25 * torch.rand(N, generator=g)).to(DEV)
    leaves = [x.detach().clone(memory_format=torch.preserve_format).requires_grad_()
              for x in (X, W)]
    c = None if bias is None else bias.detach().clone().requires_grad_()
    loss, logZ = F.linear_cross_entropy(leaves[0], leaves[1], t, c, reduction="none",
                                        return_logZ=True, **kw)
    ref = R.xent(X.reshape(-1, X.shape[-1]), W, t.reshape(-1), bias, w=w, dlogZ=z, **{
        k.replace("ignore_index", "ignore"): v for k, v in kw.items()})
    R.assert_within(loss.detach().reshape(-1), ref["loss"], ref["e_loss"], "loss")
    R.assert_within(logZ.detach().reshape(-1), ref["logZ"], ref["e_logZ"], "logZ")
    if wantgrad:
        ((loss.reshape(-1) * w).sum() + (logZ.reshape(-1) * z).sum()).backward()
        assert leaves[0].grad.dtype == X.dtype and leaves[1].grad.dtype == W.dtype
        R.assert_within(leaves[0].grad.reshape(-1, X.shape[-1]), ref["dX"], ref["e_dX"], "dX")
        R.assert_within(leaves[1].grad, ref["dW"], ref["e_dW"], "dW")
        if c is not None:
            R.assert_within(c.grad, ref["dbias"], ref["e_dbias"], "dbias")
    return loss.detach(), logZ.detach(), leaves[0].grad, leaves[1].grad


# N, V, D: one row, odd sizes, edges of the 64/128/256 tiles and one past them
SHAPES = [(1, 1, 1), (1, 1000, 64), (3, 7, 5), (8, 900, 516), (9, 333, 130), (16, 6001, 515),
          (17, 600, 64), (37, 501, 103), (128, 256, 64), (129, 257, 65),
          (255, 300, 128), (257, 1024, 72), (300, 4099, 200), (513, 130, 1000), (700, 2049, 256)]


@pytest.mark.parametrize("dtype", [BF, FH, FS], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,V,D", SHAPES)
def test_xent_matches_64_bits(N, V, D, dtype):
    X, W, t, c = R.problem(N, V, D, dtype, seed=N + V + D, ignored=0.2 if N > 30 else 0,
                           bias=(N + D) % 2 == 1)
    check_xent(X, W, t, c)


@pytest.mark.parametrize("dtype", [BF, FH, FS], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,V,D", [(5, 70001, 96), (2500, 9001, 320), (9000, 600, 64),
                                   (6000, 12300, 40)])
def test_xent_larger(N, V, D, dtype):
    X, W, t, c = R.problem(N, V, D, dtype, seed=7, ignored=0.3, bias=True)
    check_xent(X, W, t, c)


@pytest.mark.parametrize("dtype", [BF, FS], ids=["bf16", "fp32"])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
def test_xent_reductions(reduction, dtype):
    X, W, t, c = R.problem(333, 555, 88, dtype, ignored=0.25, bias=True)
    X.requires_grad_(), W.requires_grad_(), c.requires_grad_()
    loss = F.linear_cross_entropy(X, W, t, c, reduction=reduction)
    assert loss.shape == () and loss.dtype == torch.float32
    (3.0 * loss).backward()
    count = int((t != R.IGNORE).sum())
    w = torch.full((333,), 3.0 / (count if reduction == "mean" else 1.0), device=DEV)
    ref = R.xent(X, W, t, c, w=w)
    scale = count if reduction == "mean" else 1.0
    R.assert_within(loss.detach(), ref["loss"].sum() / scale,
                    ref["e_loss"].sum() / scale + 2 ** -23 * ref["loss"].sum() / scale, "loss")
    for got, name in ((X.grad, "dX"), (W.grad, "dW"), (c.grad, "dbias")):
        R.assert_within(got, ref[name], ref["e_" + name] * (1 + 2 ** -20)
                        + 2 ** -22 * ref[name].abs(), name)


def test_xent_leading_dimensions_and_int32_targets():
    X, W, t, _ = R.problem(60, 200, 40, BF)
    a = F.linear_cross_entropy(X.view(3, 20, 40), W, t.view(3, 20).int(), reduction="none")
    b = F.linear_cross_entropy(X, W, t, reduction="none")
    assert a.shape == (3, 20) and torch.equal(a.reshape(-1), b)
    one = F.linear_cross_entropy(X[0], W, t[0], reduction="none")
    assert one.shape == () and abs((one - b[0]).item()) <= 1e-5 * max(1.0, float(b[0]))


@pytest.mark.parametrize("N", [5, 13, 150])
@pytest.mark.parametrize("dtype", [BF, FS], ids=["bf16", "fp32"])
@pytest.mark.parametrize("layout", ["transposed W", "transposed X", "odd row stride",
                                    "column step", "offset base", "expanded X"])
def test_xent_strides(layout, dtype, N):
    X, W, t, c = R.problem(N, 333, 48, dtype, bias=True, seed=3)
    if layout == "transposed W":
        W = W.t().contiguous().t()
    elif layout == "transposed X":
        X = X.t().contiguous().t()
    elif layout == "odd row stride":
        X = torch.cat([X, X[:, :3]], 1)[:, :48]
        W = torch.cat([W, W[:, :5]], 1)[:, :48]
    elif layout == "column step":
        X = torch.stack([X, X * 0 + 9], 2).reshape(N, 96)[:, ::2]
        W = torch.stack([W, W * 0 + 9], 2).reshape(333, 96)[:, ::2]
    elif layout == "offset base":
        X = torch.cat([X.new_zeros(1), X.reshape(-1)])[1:].view(N, 48)
        W = torch.cat([W.new_zeros(1), W.reshape(-1)])[1:].view(333, 48)
    else:
        X = X[:1].expand(N, 48)
    Xl, Wl, cl = X.detach().requires_grad_(), W.detach().requires_grad_(), c.requires_grad_()
    assert Xl.stride() == X.stride() and Wl.stride() == W.stride()
    w = torch.rand(N, device=DEV) + 0.5
    loss = F.linear_cross_entropy(Xl, Wl, t, cl, reduction="none")
    got = torch.autograd.grad((loss * w).sum(), (Xl, Wl, cl))
    ref = R.xent(X, W, t, c, w=w)
    R.assert_within(loss.detach(), ref["loss"], ref["e_loss"], "loss")
    for x, name in zip(got, ("dX", "dW", "dbias")):
        R.assert_within(x, ref[name], ref["e_" + name], name)


@pytest.mark.parametrize("dtype", [BF, FH, FS], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("V,D,layout", [
    (1, 1, "rows"), (7, 3, "rows"), (9, 511, "rows"), (1003, 513, "rows"), (64, 129, "rows"),
    (20001, 1025, "rows"), (333, 516, "rows"), (300, 200, "transposed"), (5001, 77, "transposed"),
    (300, 64, "column step"), (401, 100, "offset base")])
def test_xent_one_row(V, D, layout, dtype):
    """One row, W in layouts that are read in place only by the plain loads."""
    X, W, t, c = R.problem(1, V, D, dtype, bias=True, seed=V)
    if layout == "transposed":
        W = W.t().contiguous().t()
    elif layout == "column step":
        W = torch.stack([W, W * 0 + 9], 2).reshape(V, 2 * D)[:, ::2]
    elif layout == "offset base":
        W = torch.cat([W.new_zeros(1), W.reshape(-1)])[1:].view(V, D)
    if V > 8:
        c[(t + 1) % V] = float("-inf")
    Xl, Wl, cl = X.requires_grad_(), W.detach().requires_grad_(), c.requires_grad_()
    assert Wl.stride() == W.stride() and Wl.data_ptr() == W.data_ptr()
    loss, logZ = F.linear_cross_entropy(Xl, Wl, t, cl, reduction="none", return_logZ=True)
    ref = R.xent(X, W, t, c, w=torch.ones(1, device=DEV), dlogZ=torch.ones(1, device=DEV))
    R.assert_within(loss.detach(), ref["loss"], ref["e_loss"], "loss")
    R.assert_within(logZ.detach(), ref["logZ"], ref["e_logZ"], "logZ")
    got = torch.autograd.grad(loss.sum() + logZ.sum(), (Xl, Wl, cl), retain_graph=True)
    again = torch.autograd.grad(loss.sum() + logZ.sum(), (Xl, Wl, cl))
    for x, y, name in zip(got, again, ("dX", "dW", "dbias")):
        R.assert_within(x, ref[name], ref["e_" + name], name)
        assert torch.equal(x, y)
    # some gradients only; an ignored row; a label outside the table
    loss = F.linear_cross_entropy(X.detach(), W.detach(), t, cl, reduction="sum")
    ref = R.xent(X, W, t, c, w=torch.ones(1, device=DEV))
    R.assert_within(torch.autograd.grad(loss, cl)[0], ref["dbias"], ref["e_dbias"], "dbias")
    off = F.linear_cross_entropy(Xl, Wl, torch.full_like(t, R.IGNORE), cl, reduction="sum")
    assert off.item() == 0.0 and not any(g.any() for g in torch.autograd.grad(off, (Xl, Wl, cl)))
    bad = F.linear_cross_entropy(Xl, Wl, torch.full_like(t, V), cl, reduction="sum")
    assert math.isnan(bad.item())
    assert all(bool(torch.isnan(g).all()) for g in torch.autograd.grad(bad, (Xl, Wl)))


@pytest.mark.parametrize("dtype", [BF, FH, FS], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N", [7, 16, 100, 300])
def test_xent_ignored_rows_may_hold_anything(N, dtype):
    X, W, t, c = R.problem(N, 400, 72, dtype, ignored=0.4, bias=True)
    dead = t == R.IGNORE
    assert 0 < int(dead.sum()) < N
    X[dead] = float("nan")
    X[dead.nonzero()[0]] = float("inf")
    X.requires_grad_(), W.requires_grad_(), c.requires_grad_()
    loss, logZ = F.linear_cross_entropy(X, W, t, c, reduction="none", return_logZ=True)
    assert not loss[dead].any() and not logZ[dead].any()
    loss.sum().backward()
    ref = R.xent(X, W, t, c, w=torch.ones(N, device=DEV))
    R.assert_within(loss.detach(), ref["loss"], ref["e_loss"], "loss")
    assert not X.grad[dead].any()
    for got, name in ((X.grad, "dX"), (W.grad, "dW"), (c.grad, "dbias")):
        R.assert_within(got, ref[name], ref["e_" + name], name)


@pytest.mark.parametrize("N", [0, 5, 300])
def test_xent_no_live_rows(N):
    X = torch.full((N, 24), float("nan"), device=DEV, dtype=BF, requires_grad=True)
    W = torch.randn(50, 24, device=DEV).to(BF).requires_grad_()
    c = torch.zeros(50, device=DEV, requires_grad=True)
    t = torch.full((N,), R.IGNORE, device=DEV)
    assert math.isnan(F.linear_cross_entropy(X, W, t, c).item())
    loss = F.linear_cross_entropy(X, W, t, c, reduction="sum")
    assert loss.item() == 0.0
    loss.backward()
    for g in (X.grad, W.grad, c.grad):
        assert not g.any()
    mean = F.linear_cross_entropy(X, W, t, c)
    for g in torch.autograd.grad(mean, (X, W, c)):
        assert not g.any()


@pytest.mark.parametrize("dtype", [BF, FS], ids=["bf16", "fp32"])
@pytest.mark.parametrize("N", [6, 14, 70, 400])
def test_xent_label_outside_the_table_is_nan(N, dtype):
    X, W, t, _ = R.problem(N, 300, 32, dtype)
    t[3], t[N - 1] = 300, -7
    X.requires_grad_(), W.requires_grad_()
    loss = F.linear_cross_entropy(X, W, t, reduction="none")
    bad = torch.zeros(N, dtype=torch.bool, device=DEV)
    bad[3] = bad[N - 1] = True
    assert torch.equal(torch.isnan(loss), bad)
    loss.sum().backward()
    assert torch.equal(torch.isnan(X.grad).any(1), bad) and bool(torch.isnan(W.grad).all())


def test_xent_ignore_index_inside_the_table():
    X, W, t, c = R.problem(90, 40, 16, FH, bias=True)
    check_xent(X, W, t % 4, c, ignore_index=2)


@pytest.mark.parametrize("dtype", [BF, FS], ids=["bf16", "fp32"])
def test_xent_removed_entries(dtype):
    X, W, t, c = R.problem(140, 700, 64, dtype, bias=True)
    gone = torch.zeros(700, dtype=torch.bool, device=DEV)
    gone[200:650] = True                 # whole tiles of the vocabulary among it
    gone[t] = False
    c[gone] = float("-inf")
    _, _, _, dW = check_xent(X, W, t, c)
    assert not dW[gone].any()
    # the type's lowest value instead of -inf: the same removal, without a NaN
    lowest = torch.where(gone, torch.full_like(c, torch.finfo(torch.float32).min), c)
    a = F.linear_cross_entropy(X, W, t, lowest, reduction="none")
    b = F.linear_cross_entropy(X, W, t, c, reduction="none")
    assert torch.equal(a, b)


def test_xent_every_entry_removed():
    X, W, t, c = R.problem(9, 300, 16, BF, bias=True)
    c[:] = float("-inf")
    loss, logZ = F.linear_cross_entropy(X, W, t, c, reduction="none", return_logZ=True)
    assert bool((logZ == -math.inf).all()) and bool(torch.isnan(loss).all())
    c[:] = torch.finfo(torch.float32).min    # all equal: a uniform distribution, up to fp32 steps
    loss, logZ = F.linear_cross_entropy(X, W, t, c, reduction="none", return_logZ=True)
    assert bool((logZ == torch.finfo(torch.float32).min).all()) and not loss.any()


@pytest.mark.parametrize("dtype", [BF, FH, FS], ids=["bf16", "fp16", "fp32"])
def test_xent_large_logits(dtype):
    """Logits of several hundred: exp alone would overflow; peaked rows."""
    X, W, t, _ = R.problem(64, 500, 64, dtype, spread=60.0)
    check_xent(X, W, t)


def test_xent_small_and_uneven_weights():
    """fp16 gradients of weights that span 2^-20 .. 1 within one call."""
    X, W, t, _ = R.problem(200, 300, 32, FH)
    X.requires_grad_(), W.requires_grad_()
    w = torch.exp2(-20 * torch.rand(200, device=DEV))
    (F.linear_cross_entropy(X, W, t, reduction="none") * w).sum().backward()
    ref = R.xent(X, W, t, None, w=w)
    R.assert_within(X.grad, ref["dX"], ref["e_dX"], "dX")
    R.assert_within(W.grad, ref["dW"], ref["e_dW"], "dW")


def test_xent_gradient_by_differences():
    X, W, t, c = R.problem(20, 60, 24, FS, bias=True, seed=5)
    X.requires_grad_(), W.requires_grad_(), c.requires_grad_()
    F.linear_cross_entropy(X, W, t, c, reduction="sum").backward()
    h = 2.0 ** -6
    for leaf in (X, W, c):
        U = torch.randn_like(leaf)
        U /= U.norm()
        old = leaf.data.clone()
        leaf.data = old + h * U
        up = F.linear_cross_entropy(X, W, t, c, reduction="sum").item()
        leaf.data = old - h * U
        down = F.linear_cross_entropy(X, W, t, c, reduction="sum").item()
        leaf.data = old
        # sums of 20 losses below 2^8 are off by at most 2^-17 each way; the difference
        # quotient by h^2 times a third derivative, which a step of norm 1 in logits of
        # rows |x|, |w| < 16 keeps below 16^3 / 6 on its few rows
        assert abs((up - down) / (2 * h) - float((leaf.grad * U).sum())) \
            <= 2.0 ** -17 / h + h * h * 16 ** 3 / 6


def test_xent_only_what_is_asked():
    X, W, t, c = R.problem(50, 80, 16, BF, bias=True)
    for k in range(3):
        leaves = [x.detach().clone().requires_grad_(i == k) for i, x in enumerate((X, W, c))]
        F.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2]).backward()
        assert [x.grad is not None for x in leaves] == [i == k for i in range(3)]
    with torch.no_grad():
        assert not F.linear_cross_entropy(X, W, t, c).requires_grad


def test_xent_same_bits_every_run():
    X, W, t, c = R.problem(6000, 12300, 136, BF, ignored=0.1, bias=True)
    X.requires_grad_(), W.requires_grad_(), c.requires_grad_()
    runs = []
    for _ in range(3):
        loss = F.linear_cross_entropy(X, W, t, c)
        runs.append((loss.detach(), *torch.autograd.grad(loss, (X, W, c))))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_xent_other_stream_and_two_at_once():
    X, W, t, _ = R.problem(500, 3000, 128, BF)
    X2, W2, t2, _ = R.problem(400, 2500, 96, BF, seed=9)
    want, want2 = (F.linear_cross_entropy(*p, reduction="none") for p in ((X, W, t), (X2, W2, t2)))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            a = F.linear_cross_entropy(X, W, t, reduction="none")
        with torch.cuda.stream(s2):
            b = F.linear_cross_entropy(X2, W2, t2, reduction="none")
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want2)


def test_backward_calls_on_two_streams_at_once():
    """Each call's pairs of SMs wait for one another; two calls share the SMs."""
    probs = [R.problem(2500, 9000, 128, BF, seed=k, bias=True) for k in (0, 1)]
    args = []
    for X, W, t, c in probs:
        loss, logZ, _, count = L.xent_fwd(X, W, t, c, R.IGNORE, "mean")
        args.append((X, W, t, c, R.IGNORE, logZ, torch.ones((), device=DEV), count, None,
                     (True, True, True)))
    want = [L.xent_bwd(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(L.xent_bwd(*args[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        for out in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[k]))


@pytest.mark.parametrize("dtype", [BF, FS], ids=["bf16", "fp32"])
def test_xent_mean_with_a_penalty_on_logz(dtype):
    X, W, t, c = R.problem(400, 900, 56, dtype, ignored=0.2, bias=True, seed=4)
    leaves = [x.clone().requires_grad_() for x in (X, W, c)]
    loss, logZ = F.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], return_logZ=True)
    (loss + 1e-3 * logZ.square().sum()).backward()
    count = int((t != R.IGNORE).sum())
    w = torch.full((400,), 1.0 / count, device=DEV)
    z = R.xent(X, W, t, c)["logZ"] * 2e-3
    ref = R.xent(X, W, t, c, w=w, dlogZ=z)
    # the penalty's weight is made of the float32 logZ: 2^-17 + 2^-22 of it at most (e_logZ)
    off = 2e-3 * ref["e_logZ"].max() / z.abs().max().clamp_min(1e-6) + 2 ** -20
    for leaf, name in zip(leaves, ("dX", "dW", "dbias")):
        slack = off * {"dX": (z + 1)[:, None] * W.double().abs().max(),
                       "dW": (z.abs().sum() + 1) * X.double().abs().max(),
                       "dbias": z.abs().sum() + 1}[name]
        R.assert_within(leaf.grad, ref[name], ref["e_" + name] * (1 + 2 ** -18) + slack, name)


@pytest.mark.parametrize("N", [255, 256, 257])
def test_xent_rows_read_in_place_or_copied(N):
    """Up to 256 16-bit rows are read in place, with their ignored rows among them."""
    X, W, t, _ = R.problem(N, 5000, 96, BF, ignored=0.3, seed=N)
    wide = torch.cat([X, X], 1)
    X[t == R.IGNORE] = float("nan")
    wide[t == R.IGNORE] = float("nan")
    a = F.linear_cross_entropy(X, W, t, reduction="none")
    b = F.linear_cross_entropy(wide[:, 96:], W, t, reduction="none")
    c = F.linear_cross_entropy(wide[:, 96:].contiguous()[:, :], W, t, reduction="sum")
    ref = R.xent(X.nan_to_num(0), W, t, None)
    R.assert_within(a, ref["loss"], ref["e_loss"], "loss")
    assert torch.equal(a, b)
    assert abs(c.item() - ref["loss"].sum().item()) <= ref["e_loss"].sum().item() + 2 ** -20 * c.item()


def test_xent_from_new_host_threads():
    """The backward call as the first CUDA call of its host thread (as autograd's worker
    makes it), and two threads on one stream at once."""
    import threading
    X, W, t, _ = R.problem(300, 500, 64, BF)
    loss, logZ, reduced, count = L.xent_fwd(X, W, t, None, R.IGNORE, "mean")
    one = torch.ones((), device=DEV)
    want = L.xent_bwd(X, W, t, None, R.IGNORE, logZ, one, count, None, (True, True, False))
    got, failed = {}, []

    def work(k):
        try:
            for _ in range(10):
                got[k] = L.xent_bwd(X, W, t, None, R.IGNORE, logZ, one, count, None,
                                    (True, True, False))
                assert torch.equal(L.xent_fwd(X, W, t, None, R.IGNORE, "none")[0], loss)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    [th.start() for th in threads]
    [th.join() for th in threads]
    assert not failed, failed
    for g in got.values():
        assert torch.equal(g[0], want[0]) and torch.equal(g[1], want[1])


def test_training_step_captured_into_graphs():
    """Lookup, loss and both gradients, captured twice and replayed on new data."""
    X, W, t, _ = R.problem(300, 700, 64, BF, ignored=0.1)
    ids = torch.randint(0, 700, (300,), device=DEV)

    def step(X, W, t, ids):
        rows = F.embedding_lookup(W, ids, scale=8.0)
        loss = F.linear_cross_entropy(X + rows, W, t)
        return loss.detach(), *torch.autograd.grad(loss, (X, W))

    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):
        a = [X.detach().clone().requires_grad_(), W.detach().clone().requires_grad_(), t.clone(),
             ids.clone()]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*a)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*a)
        graphs.append((g, a, out))
    for k, (g, a, out) in enumerate(graphs):
        with torch.no_grad():
            a[0].copy_(X.flip(0) if k else X * 0.5)
            a[2].copy_(t.flip(0) if k else t)
    for g, _, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, a, out in graphs:
        want = step(*[x.detach().clone().requires_grad_(x.is_floating_point()) for x in a])
        assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_tied_table_step():
    """Lookup, loss, and both ends' gradients of one table added in place."""
    V, D, N = 900, 80, 350
    X, W, t, _ = R.problem(N, V, D, FS, ignored=0.1)
    ids = torch.randint(0, V, (N,), device=DEV)
    W.requires_grad_()
    rows = F.embedding_lookup(W, ids, scale=0.5)
    h = (rows + X).detach().requires_grad_()
    loss = F.linear_cross_entropy(h, W, t)
    dh, dW = torch.autograd.grad(loss, (h, W))
    total = F.embedding_grad(dh, ids, V, scale=0.5, out=dW.clone(), accumulate=True)
    # the same through autograd, both ends at once
    loss2 = F.linear_cross_entropy(F.embedding_lookup(W, ids, scale=0.5) + X, W, t)
    auto, = torch.autograd.grad(loss2, W)
    extra, bound = R.embed_grad(dh, ids, V, 0.5)
    assert torch.equal(loss, loss2)
    want = dW.double() + extra
    R.assert_within(total, want, bound + 2 ** -23 * (want.abs() + dW.double().abs()), "tied")
    R.assert_within(auto, want, bound + 2 ** -22 * (want.abs() + dW.double().abs()), "autograd")


def test_xent_logz_is_the_estep():
    """W = mu, bias = log pi - |mu|^2/2: logZ and the gradients of its sum are the
    isotropic E-step's logZ, mu_acc and Nk at unit variance."""
    g = torch.Generator().manual_seed(2)
    N, K, D = 3000, 200, 48
    mu = torch.randn(K, D, generator=g).to(DEV)
    X = (mu[torch.randint(0, K, (N,), generator=g).to(DEV)]
         + torch.randn(N, D, generator=g).to(DEV))
    lpi = torch.log_softmax(torch.randn(K, generator=g), 0).to(DEV)
    logZ, Nk, mu_acc, _ = flash_gmm.flash_gmm_estep(X, mu, torch.zeros(K, device=DEV), lpi)
    W = mu.clone().requires_grad_()
    c = (lpi - 0.5 * mu.double().square().sum(1)).float().requires_grad_()
    t = torch.zeros(N, dtype=torch.int64, device=DEV)
    _, z = F.linear_cross_entropy(X, W, t, c, reduction="none", return_logZ=True)
    shift = 0.5 * X.double().square().sum(1) + 0.5 * D * math.log(2 * math.pi)
    off = ((z.detach().double() - shift) - logZ.double()).abs().max()
    # each side is held to 1e-5 of max(1, |logZ|); z is |x|^2/2 larger at most
    assert off.item() <= 1e-5 * (logZ.abs().max().item() + shift.max().item())
    z.sum().backward()
    for got, want in ((W.grad, mu_acc), (c.grad, Nk)):
        assert float((got - want).abs().max()) <= 2e-4 * float(want.abs().max())


# ---------------------------------------------------------------- embedding
@pytest.mark.parametrize("dtype", [BF, FH, FS], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 1000, 64), (7, 3, 5), (300, 50, 129),
                                   (2048, 256, 72), (2049, 70000, 33), (5000, 4097, 264),
                                   (40000, 300, 16), (1500, 65536, 1000)])
def test_embedding_matches_64_bits(N, V, D, dtype):
    g = torch.Generator().manual_seed(N + V)
    table = torch.randn(V, D, generator=g).to(dtype).to(DEV).requires_grad_()
    # half of the ids from a few rows: long runs beside single ids and empty rows
    ids = torch.where(torch.rand(N, generator=g) < 0.5, torch.randint(0, min(V, 3), (N,), generator=g),
                      torch.randint(0, V, (N,), generator=g)).to(DEV)
    if N > 100:
        ids[::17] = R.IGNORE
    dout = torch.randn(N, D, generator=g).to(dtype).to(DEV)
    out = F.embedding_lookup(table, ids, scale=0.7)
    keep = (ids != R.IGNORE)[:, None]
    want = torch.where(keep, table.detach().double()[ids.clamp_min(0)] * 0.7, 0.0)
    u = R.U[dtype]
    R.assert_within(out.detach(), want, (u + 2 ** -22) * want.abs() + R.TINY[dtype], "lookup")
    out.backward(dout)
    ref, bound = R.embed_grad(dout, ids, V, 0.7)
    R.assert_within(table.grad, ref, bound, "dtable")
    again = F.embedding_grad(dout, ids, V, scale=0.7)
    assert torch.equal(again, table.grad)


@pytest.mark.parametrize("layout", ["transposed", "odd row stride", "offset base"])
def test_embedding_strides(layout):
    table, dout = torch.randn(90, 40, device=DEV), torch.randn(200, 40, device=DEV).to(BF)
    ids = torch.randint(0, 90, (200,), device=DEV)
    if layout == "transposed":
        a, d = table.t().contiguous().t(), dout.t().contiguous().t()
    elif layout == "odd row stride":
        a, d = torch.cat([table, table[:, :1]], 1)[:, :40], torch.cat([dout, dout[:, :1]], 1)[:, :40]
    else:
        a = torch.cat([table.new_zeros(1), table.reshape(-1)])[1:].view(90, 40)
        d = torch.cat([dout.new_zeros(1), dout.reshape(-1)])[1:].view(200, 40)
    assert torch.equal(F.embedding_lookup(a, ids.view(10, 20)), table[ids].view(10, 20, 40))
    assert torch.equal(F.embedding_grad(d, ids, 90), F.embedding_grad(dout, ids, 90))


def test_embedding_bad_ids():
    table = torch.randn(20, 8, device=DEV, requires_grad=True)
    ids = torch.tensor([3, 20, -1, -100, 19], device=DEV)
    out = F.embedding_lookup(table, ids)
    assert torch.isnan(out[1:3]).all() and not out[3].any()
    assert torch.equal(out[[0, 4]], table[[3, 19]])
    dtable = F.embedding_grad(torch.ones(5, 8, device=DEV), ids, 20)
    want = torch.zeros(20, 8, device=DEV)
    want[3] = want[19] = 1
    assert torch.equal(dtable, want)


def test_embedding_ignore_index_inside_the_table():
    table = torch.randn(20, 8, device=DEV, requires_grad=True)
    ids = torch.tensor([0, 5, 0, 6], device=DEV)
    out = F.embedding_lookup(table, ids, ignore_index=0)
    assert not out[[0, 2]].any()
    out.sum().backward()
    assert not table.grad[0].any() and bool((table.grad[5] == 1).all())


@pytest.mark.parametrize("dtype", [BF, FS], ids=["bf16", "fp32"])
def test_embedding_accumulate_leaves_other_rows(dtype):
    V, D, N = 500, 72, 90
    ids = torch.randint(0, 40, (N,), device=DEV)
    dout = torch.randn(N, D, device=DEV).to(dtype)
    old = torch.randn(V, D, device=DEV).to(dtype)
    old[100] = float("nan")
    got = F.embedding_grad(dout, ids, V, out=old.clone(), accumulate=True)
    assert torch.equal(got[101:], old[101:]) and bool(torch.isnan(got[100]).all())
    ref, bound = R.embed_grad(dout, ids, V, 1.0)
    want = old[:100].double() + ref[:100]
    touched = torch.bincount(ids, minlength=V)[:100, None] > 0
    R.assert_within(got[:100], want, torch.where(
        touched, bound[:100] + (R.U[dtype] + 2 ** -23) * (want.abs() + old[:100].double().abs()),
        torch.zeros_like(want)), "accumulated")


def test_embedding_empty_calls():
    table = torch.randn(20, 8, device=DEV, requires_grad=True)
    out = F.embedding_lookup(table, torch.zeros(0, 3, dtype=torch.int64, device=DEV))
    assert out.shape == (0, 3, 8)
    out.sum().backward()
    assert not table.grad.any()
    keep = torch.ones(20, 8, device=DEV)
    F.embedding_grad(torch.zeros(0, 8, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV),
                     20, out=keep, accumulate=True)
    assert bool((keep == 1).all())


def test_embedding_one_id_many_times():
    """One id 30,000 times beside a few others: the longest run and its neighbours."""
    N, D = 30011, 40
    ids = torch.full((N,), 11, device=DEV)
    ids[::1000] = torch.arange(len(ids[::1000]), device=DEV)
    dout = torch.randn(N, D, device=DEV)
    ref, bound = R.embed_grad(dout, ids, 64, 1.0)
    R.assert_within(F.embedding_grad(dout, ids, 64), ref, bound, "dtable")


def test_tables_longer_than_32_bit_offsets():
    """V * D > 2^31 elements: rows and columns at the far end."""
    V, D = 1_200_000, 2048
    table = torch.empty(V, D, device=DEV, dtype=BF)
    for i in range(0, V, 100_000):
        table[i:i + 100_000] = torch.randn(1, D, device=DEV) * 0.02
    table[V - 3:] = torch.randn(3, D, device=DEV) * 0.05
    ids = torch.tensor([V - 1, 0, V - 2, 600_000, V - 1], device=DEV)
    assert torch.equal(F.embedding_lookup(table, ids), table[ids])
    X = table[ids[:3]].float().mul(4).to(BF)
    loss, logZ = F.linear_cross_entropy(X, table, ids[:3], reduction="none", return_logZ=True)
    S = torch.cat([X.double() @ table[i:i + 100_000].double().t() for i in range(0, V, 100_000)], 1)
    want = torch.logsumexp(S, 1)
    assert float((logZ.double() - want).abs().max()) < 1e-3
    assert float((loss.double() - (want - S[[0, 1, 2], ids[:3]])).abs().max()) < 1e-3
    g = torch.randn(5, D, device=DEV).to(BF)
    d = F.embedding_grad(g, ids, V)
    assert torch.equal(d[V - 1], (g[0].float() + g[4].float()).to(BF))
    assert torch.equal(d[600_000], g[3]) and not d[V - 3].any()


def test_launches_are_the_librarys():
    before = L.launch_count()
    X, W, t, _ = R.problem(20, 30, 8, BF)
    F.linear_cross_entropy(X, W, t)
    F.embedding_lookup(W, t)
    assert L.launch_count() >= before + 3


@pytest.mark.parametrize("dtype", [FS, BF, torch.float64], ids=["fp32", "bf16", "fp64"])
def test_init_params_rows_are_unchanged(dtype):
    import gmm_em
    X = torch.randn(5000, 24, device=DEV).to(dtype)
    for Y in (X, X.t().contiguous().t()):
        mu, _, _ = gmm_em.init_params(Y, 64, seed=3)
        idx = torch.randperm(5000, generator=torch.Generator().manual_seed(3))[:64].to(DEV)
        assert mu.dtype == torch.float32 and torch.equal(mu, X[idx].float())


@pytest.mark.parametrize("dtype", [BF, FH, FS], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N", [1, 12, 300, 5000])
def test_xent_bias_gradient_without_a_bias(N, dtype):
    """The C entry takes dbias with a NULL bias: the sums of g over the rows."""
    V, D = 2999, 40
    X, W, t, _ = R.problem(N, V, D, dtype, seed=N)
    kind, lib = L.FGMM_TYPES[dtype], L.load()
    loss, logZ, _, _ = L.xent_fwd(X, W, t, None, R.IGNORE, "none")
    w = torch.rand(N, device=DEV) + 0.5
    need = lib.fgmm_xent_workspace_bytes(1, kind, N, V, D, W.data_ptr(), D, 1, 1)
    # bytes behind the stated workspace have to stay as they are
    ws = torch.full((need + (1 << 20),), 77, dtype=torch.uint8, device=DEV)
    dX, dW, dbias = torch.empty_like(X), torch.empty_like(W), torch.empty(V, device=DEV)
    L._launch(lib.fgmm_xent_bwd, X.device, kind, X.data_ptr(), D, 1, W.data_ptr(), D, 1, None,
              t.data_ptr(), R.IGNORE, N, V, D, logZ.data_ptr(), w.data_ptr(), 1, None, None,
              dX.data_ptr(), dW.data_ptr(), dbias.data_ptr(), ws.data_ptr(), need)
    assert bool((ws[need:] == 77).all())
    ref = R.xent(X, W, t, None, w=w)
    for got, name in ((dX, "dX"), (dW, "dW"), (dbias, "dbias")):
        R.assert_within(got, ref[name], ref["e_" + name], name)


@pytest.mark.parametrize("dtype,N,V,D", [(BF, 5000, 70000, 64), (FH, 9000, 9000, 33),
                                         (FS, 9000, 9000, 33)], ids=["bf16", "fp16", "fp32"])
def test_xent_gradient_over_many_pieces(dtype, N, V, D):
    """Pieces of g that go round the ring several times, sums of dX and dW handed from SM
    to SM: right, and the same bits, in every one of many runs."""
    X, W, t, _ = R.problem(N, V, D, dtype, seed=11)
    loss, logZ, _, _ = L.xent_fwd(X, W, t, None, R.IGNORE, "none")
    one = torch.ones((), device=DEV)
    call = lambda: L.xent_bwd(X, W, t, None, R.IGNORE, logZ, one, None, None, (True, True, False))
    first = call()
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(call()[:2], first[:2]))
    rows = torch.arange(0, N, 97, device=DEV)            # dX of some rows
    part = R.xent(X[rows], W, t[rows], None, w=torch.ones(len(rows), device=DEV))
    R.assert_within(first[0][rows], part["dX"], part["e_dX"], "dX")
    if V <= 10000:
        ref = R.xent(X, W, t, None, w=torch.ones(N, device=DEV))
        R.assert_within(first[1], ref["dW"], ref["e_dW"], "dW")


@pytest.mark.parametrize("bias", [False, True], ids=["plain", "bias"])
@pytest.mark.parametrize("power", [6, 9, 12])
@pytest.mark.parametrize("dtype", [BF, FS], ids=["bf16", "fp32"])
def test_xent_logits_far_beyond_the_exponentials_range(dtype, power, bias):
    """Rows as a diverged model gives them: the largest logit takes all of the probability."""
    N, V, D = 40, 500, 64
    X, W, t, c = R.problem(N, V, D, dtype, seed=power, bias=bias)
    X = X * 10.0 ** power
    X.requires_grad_(), W.requires_grad_()
    ref = R.xent(X, W, t, c)
    loss, logZ = F.linear_cross_entropy(X, W, t, c, reduction="none", return_logZ=True)
    R.assert_within(loss.detach(), ref["loss"], ref["e_loss"], "loss")
    R.assert_within(logZ.detach(), ref["logZ"], ref["e_logZ"], "logZ")
    dX, dW = torch.autograd.grad(loss.sum(), (X, W))
    # logits are known within e_logZ: where the largest leads by more than that and 200,
    # every other exponential is zero, in 64 bits and in 32
    S = X.detach().double() @ W.detach().double().t()
    top = S.topk(2, 1)
    sure = top.values[:, 0] - top.values[:, 1] > 2 * ref["e_logZ"] + 200
    assert int(sure.sum()) > N // 2
    G = torch.zeros(N, V, device=DEV, dtype=torch.float64)
    rows = torch.arange(N, device=DEV)
    G[rows, top.indices[:, 0]] = 1.0
    G[rows, t] -= 1.0
    u = R.U[dtype]
    want = G @ W.detach().double()
    mag = G.abs() @ W.detach().double().abs()
    R.assert_within(dX[sure], want[sure], ((u + R.chain(V)) * mag + R.TINY[dtype])[sure], "dX")
    # entries that only such rows name
    only = ((G != 0) & ~sure[:, None]).sum(0) == 0
    only &= ((S - S.amax(1, keepdim=True) > -2 * ref["e_logZ"][:, None] - 200)
             & ~sure[:, None]).sum(0) == 0
    want = G.t() @ X.detach().double()
    mag = G.abs().t() @ X.detach().double().abs()
    R.assert_within(dW[only], want[only], ((u + R.chain(N)) * mag + R.TINY[dtype])[only], "dW")


@pytest.mark.parametrize("dtype", [BF, FH, FS], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,V,D", [(27011, 5000, 16), (150000, 700, 8)])
def test_xent_bias_gradient_over_many_chunks_of_rows(N, V, D, dtype):
    """More chunks of rows than the ring has pieces: their parts of dbias add up."""
    X, W, t, c = R.problem(N, V, D, dtype, seed=12, ignored=0.1, bias=True)
    w = torch.rand(N, device=DEV) + 0.5
    parts = [R.xent(X[i:i + 30000], W, t[i:i + 30000], c, w=w[i:i + 30000])
             for i in range(0, N, 30000)]
    want, bound = (sum(p[k] for p in parts) for k in ("dbias", "e_dbias"))
    # the parts' own terms of the sum's length are for 30,000 rows each
    bound = bound + 2.0 ** -24 * (N / 32 + 64) * sum(p["dbias"].abs() for p in parts)
    for others in (False, True):
        leaves = [X.clone().requires_grad_(others), W.clone().requires_grad_(others),
                  c.clone().requires_grad_()]
        loss = F.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction="none")
        wanted = [x for x in leaves if x.requires_grad]
        got = torch.autograd.grad((loss * w).sum(), wanted, retain_graph=True)
        R.assert_within(got[-1], want, bound, "dbias")
        again = torch.autograd.grad((loss * w).sum(), wanted)
        assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_init_params_of_more_columns_than_the_lookup_takes():
    import gmm_em
    X = torch.randn(6, 65537, device=DEV)
    mu, _, _ = gmm_em.init_params(X, 3, seed=1)
    idx = torch.randperm(6, generator=torch.Generator().manual_seed(1))[:3].to(DEV)
    assert torch.equal(mu, X[idx])


@pytest.mark.parametrize("dtype", [FS, BF], ids=["fp32", "bf16"])
def test_init_params_passes_derivatives_to_its_rows(dtype):
    import gmm_em
    X = torch.randn(50, 24, device=DEV).to(dtype).requires_grad_()
    idx = torch.randperm(50, generator=torch.Generator().manual_seed(1))[:7].to(DEV)
    mu, _, _ = gmm_em.init_params(X, 7, seed=1)
    g = torch.randn(7, 24, device=DEV)
    want = torch.zeros(50, 24, device=DEV, dtype=dtype)
    want[idx] = g.to(dtype)
    assert torch.equal(torch.autograd.grad(mu, X, g)[0], want)
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        tangent = torch.randn(50, 24, device=DEV).to(dtype)
        mu, _, _ = gmm_em.init_params(fw.make_dual(X.detach(), tangent), 7, seed=1)
        assert torch.equal(fw.unpack_dual(mu).tangent, tangent[idx].float())


def test_embedding_grad_into_a_buffer_is_seen_by_autograd():
    ids, dout = torch.randint(0, 20, (30,), device=DEV), torch.randn(30, 8, device=DEV)
    out = torch.randn(20, 8, device=DEV)
    for accumulate in (False, True):
        a = torch.randn(20, 8, device=DEV, requires_grad=True)
        product = (a * out).sum()          # saves out for a's gradient
        before = out._version
        F.embedding_grad(dout, ids, 20, out=out, accumulate=accumulate)
        assert out._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.backward()
    with torch.inference_mode():
        F.embedding_grad(dout, ids, 20, out=torch.zeros(20, 8, device=DEV), accumulate=True)


def negated(x):
    """x's values as the imaginary part of a conjugate: a view whose memory holds -x."""
    z = torch.complex(torch.zeros_like(x), -x).conj().imag
    assert z.is_neg() and torch.equal(z, x)
    return z


@pytest.mark.parametrize("N", [5, 50])
def test_negated_views_have_their_values(N):
    X, W, t, c = R.problem(N, 90, 24, FS, bias=True)
    w = torch.rand(N, device=DEV) + 0.5

    def grads(X, W, c, w):
        leaves = [x.detach().requires_grad_() for x in (X, W, c)]
        assert [x.is_neg() for x in leaves] == [x.is_neg() for x in (X, W, c)]
        loss, logZ = F.linear_cross_entropy(*leaves[:2], t, leaves[2], reduction="none",
                                            return_logZ=True)
        return loss.detach(), *torch.autograd.grad((loss, logZ), leaves, (w, w))

    want = grads(X, W, c, w)
    for mask in range(1, 16):
        args = [negated(x) if mask >> i & 1 else x for i, x in enumerate((X, W, c, w))]
        for got, ref in zip(grads(*args), want):
            # a W of two floats' steps is summed in another order: both within 2^-18
            assert float((got - ref).abs().max()) <= 2.0 ** -18 * float(ref.abs().max().clamp_min(1))
    table = W.detach()
    assert torch.equal(F.embedding_lookup(negated(table), t), table[t])
    dout = torch.randn(N, 24, device=DEV)
    leaf = table.clone().requires_grad_()
    got, = torch.autograd.grad(F.embedding_lookup(leaf, t), leaf, negated(dout))
    assert torch.equal(got, F.embedding_grad(dout, t, 90))
    assert torch.equal(F.embedding_grad(negated(dout), t, 90), got)
    import gmm_em
    mu, _, _ = gmm_em.init_params(negated(table), 5, seed=1)
    assert torch.equal(mu, gmm_em.init_params(table, 5, seed=1)[0])


@pytest.mark.parametrize("dtype", [BF, FH], ids=["bf16", "fp16"])
def test_xent_probabilities_of_the_longest_rows(dtype):
    """D = 65536 and logits near 800, all products positive: the gradient's logits may not
    be cut more than those of logZ."""
    N, V, D = 70, 40, 65536
    g = torch.Generator().manual_seed(4)
    X = (0.5 + torch.rand(N, D, generator=g)).to(dtype).to(DEV)
    W = (800.0 / D * (1 + 0.5 * torch.randn(V, D, generator=g)).abs()).to(dtype).to(DEV)
    X.requires_grad_(), W.requires_grad_()
    t = torch.zeros(N, dtype=torch.int64, device=DEV)
    logZ = F.linear_cross_entropy(X, W, t, reduction="none", return_logZ=True)[1]
    dX, dW = torch.autograd.grad(logZ.sum(), (X, W))
    Xd, Wd = X.detach().double(), W.detach().double()
    S = Xd @ Wd.t()
    p = torch.softmax(S, 1)
    # a group of 64 steps cuts 2^-22 of its own sum a step (8 more for joining), forward 16;
    # the groups are added at 2^-24 of the sum so far each
    e = S.max() * (2.0 ** -22 * (64 + 8 + 16 + 8) + 2.0 ** -24 * (D / 1024 + D / 256)) + 2.0 ** -16
    u = R.U[dtype]
    relative = torch.expm1(e) + 2 * u + R.chain(max(V, N))     # g's and the result's rounding
    assert 2.0 ** -7 < float(relative) < 0.06
    for got, want in ((dX, p @ Wd), (dW, p.t() @ Xd)):
        R.assert_within(got, want, relative * want + R.TINY[dtype], "gradient")


@pytest.mark.parametrize("V", [200, 5000, 70001], ids=["1 pass", "2 passes", "3 passes"])
@pytest.mark.parametrize("N", [16385, 65536, 65537, 131072, 131073, 300001])
@pytest.mark.parametrize("dtype", [BF, FS], ids=["bf16", "fp32"])
def test_embedding_of_many_ids(N, V, dtype):
    """Each form of the sort: one cluster with 2, 8 and 16 ids a thread, and the long one."""
    D = 11
    g = torch.Generator().manual_seed(N + V)
    ids = torch.where(torch.rand(N, generator=g) < 0.3, torch.randint(0, 3, (N,), generator=g),
                      torch.randint(0, V, (N,), generator=g)).to(DEV)
    ids[::13] = R.IGNORE
    ids[5], ids[N - 1] = V, -1                     # outside the table
    table = torch.randn(V, D, generator=g).to(dtype).to(DEV).requires_grad_()
    dout = torch.randn(N, D, generator=g).to(dtype).to(DEV)
    out = F.embedding_lookup(table, ids)
    valid = (ids >= 0) & (ids < V)
    assert torch.equal(out[valid].detach(), table.detach()[ids[valid]])
    assert bool(torch.isnan(out[5]).all() & torch.isnan(out[N - 1]).all())
    assert not out.detach()[ids == R.IGNORE].any()
    got, = torch.autograd.grad(out, table, dout)
    ref, bound = R.embed_grad(dout, ids, V, 1.0)
    R.assert_within(got, ref, bound, "dtable")
    assert torch.equal(F.embedding_grad(dout, ids, V), got)
    # every position counted once: whole sums are exact
    ones = F.embedding_grad(torch.ones(N, D, device=DEV), ids, V)
    assert torch.equal(ones, torch.bincount(ids[valid], minlength=V)[:, None].float().expand(V, D))


@pytest.mark.parametrize("dtype", [BF, FH, FS], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N", [16384, 16385, 20480, 40001])
def test_xent_lists_long_batches(N, dtype):
    """Live rows counted in blocks of 4096 before they are listed, blocks without any among
    them; each row's loss and gradient at its own place."""
    V, D = 90, 24
    X, W, t, c = R.problem(N, V, D, dtype, seed=N, ignored=0.4, bias=True)
    t[4096:8192] = R.IGNORE
    t[9000:12500] = R.IGNORE
    X[t == R.IGNORE] = float("nan")
    X.requires_grad_(), W.requires_grad_(), c.requires_grad_()
    w = torch.rand(N, device=DEV) + 0.5
    loss, logZ = F.linear_cross_entropy(X, W, t, c, reduction="none", return_logZ=True)
    ref = R.xent(X, W, t, c, w=w)
    R.assert_within(loss.detach(), ref["loss"], ref["e_loss"], "loss")
    R.assert_within(logZ.detach(), ref["logZ"], ref["e_logZ"], "logZ")
    got = torch.autograd.grad((loss * w).sum(), (X, W, c))
    for x, name in zip(got, ("dX", "dW", "dbias")):
        R.assert_within(x, ref[name], ref["e_" + name], name)
    assert not got[0][t == R.IGNORE].any()
    mean = F.linear_cross_entropy(X, W, t, c)
    live = int((t != R.IGNORE).sum())
    R.assert_within(mean.detach(), ref["loss"].sum() / live,
                    (ref["e_loss"].sum() + 2 ** -23 * ref["loss"].sum()) / live, "mean")


def test_xent_gradient_of_a_table_longer_than_32_bit_offsets():
    """V * D > 2^31 elements in W and dW: entries at both ends and between."""
    N, V, D = 40, 1_200_000, 2048
    W = torch.empty(V, D, device=DEV, dtype=BF)
    for i in range(0, V, 100_000):
        W[i:i + 100_000] = torch.randn(1, D, device=DEV) * 0.02
    some = torch.cat([torch.arange(5), torch.arange(600_000, 600_005), torch.arange(V - 5, V)])
    some = some.to(DEV)
    W[some] = (torch.randn(15, D, device=DEV) * 0.05).to(BF)
    t = some[torch.arange(N, device=DEV) % 15]
    X = (W[t].float() * 4 + 0.1 * torch.randn(N, D, device=DEV)).to(BF)
    X.requires_grad_(), W.requires_grad_()
    loss, logZ = F.linear_cross_entropy(X, W, t, reduction="none", return_logZ=True)
    dX, dW = torch.autograd.grad(loss.sum(), (X, W))
    Xd, lz = X.detach().double(), torch.empty(N, V, device=DEV, dtype=torch.float64)
    for i in range(0, V, 100_000):
        lz[:, i:i + 100_000] = Xd @ W.detach()[i:i + 100_000].double().t()
    # all of one logit's products at once: steps of 16 that cut 2^-22 of the sum of magnitudes
    e = float(R.chain(D) * (Xd.abs() @ W.detach()[some].double().abs().t()).max()) * 2
    S, lz = lz, torch.logsumexp(lz, 1)
    assert float((logZ.detach().double() - lz).abs().max()) <= e + 2.0 ** -12
    G = torch.exp(S - lz[:, None])
    G[torch.arange(N, device=DEV), t] -= 1.0
    relative = math.expm1(2 * e + 2.0 ** -12) + 2.0 ** -8 + R.chain(V)
    want = torch.zeros(N, D, device=DEV, dtype=torch.float64)
    mag = torch.zeros_like(want)
    for i in range(0, V, 100_000):
        w = W.detach()[i:i + 100_000].double()
        want += G[:, i:i + 100_000] @ w
        mag += G[:, i:i + 100_000].abs() @ w.abs()
    # a label's p - 1 carries p's error, not that of its difference
    mag += W.detach()[t].double().abs()
    R.assert_within(dX, want, relative * mag + 2.0 ** -8 * want.abs(), "dX")
    for rows in (some, torch.tensor([99_999, 100_000, 1_048_575, 1_048_576], device=DEV)):
        g = G[:, rows]
        mag = (g.abs() + (t[:, None] == rows).double()).t() @ Xd.abs()
        R.assert_within(dW[rows], g.t() @ Xd, relative * mag + 2.0 ** -8 * (g.t() @ Xd).abs()
                        + R.TINY[BF], "dW")
