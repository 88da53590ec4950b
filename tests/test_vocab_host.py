"""The vocabulary operators' refusals, without a GPU: argument checks of
flash_vocab and of the C entries (validated before any device call)."""

import ctypes
import os

import pytest
import torch

import _fgmm_lib as L
import flash_vocab as F
import vocab_ref as R

X, W, T = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(L.LIB_PATH):
        import build_lib
        build_lib.build()
    return L.load()


@pytest.mark.parametrize("call,match", [
    (lambda: F.linear_cross_entropy(X, W, T), "must be on GPU"),
    (lambda: F.linear_cross_entropy(X, W, T, reduction="avg"), "reduction"),
    (lambda: F.linear_cross_entropy(X, torch.zeros(5, 7), T), r"X must be \(\.\.\., D\)"),
    (lambda: F.linear_cross_entropy(X, torch.zeros(8), T), r"W \(V, D\)"),
    (lambda: F.linear_cross_entropy(torch.tensor(1.0), W, T), r"X must be"),
    (lambda: F.linear_cross_entropy(X, torch.zeros(0, 8), T), "must not be empty"),
    (lambda: F.linear_cross_entropy(torch.zeros(4, 0), torch.zeros(5, 0), T), "must not be empty"),
    (lambda: F.linear_cross_entropy(X, W, T[:3]), r"targets must be \(4,\)"),
    (lambda: F.linear_cross_entropy(X, W, T.float()), "int64 or int32"),
    (lambda: F.linear_cross_entropy(X.double(), W.double(), T), "float32, bfloat16 or float16"),
    (lambda: F.linear_cross_entropy(X.bfloat16(), W, T), "one type"),
    (lambda: F.linear_cross_entropy(X, W, T, torch.zeros(4)), r"bias must be \(5,\)"),
    (lambda: F.linear_cross_entropy(X, W, T, torch.zeros(5, dtype=torch.int64)), "floating point"),
    (lambda: F.embedding_lookup(W, T), "must be on GPU"),
    (lambda: F.embedding_lookup(W[0], T), r"table must be \(V, D\)"),
    (lambda: F.embedding_lookup(W[:0], T), "not empty"),
    (lambda: F.embedding_lookup(W.double(), T), "float32, bfloat16 or float16"),
    (lambda: F.embedding_lookup(W, T.float()), "int64 or int32"),
    (lambda: F.embedding_grad(X, T, 5), "must be on GPU"),
    (lambda: F.embedding_grad(X, T[:2], 5), r"ids must be \(4,\)"),
    (lambda: F.embedding_grad(X, T, 0), "must be positive"),
    (lambda: F.embedding_grad(X, T, 5, accumulate=True), "needs the out= buffer"),
])
def test_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name,call", [
    ("linear_cross_entropy", lambda d: F.linear_cross_entropy(d(X), W, T)),
    ("linear_cross_entropy", lambda d: F.linear_cross_entropy(X, d(W), T)),
    ("linear_cross_entropy", lambda d: F.linear_cross_entropy(X, W, T, d(torch.zeros(5)))),
    ("embedding_lookup", lambda d: F.embedding_lookup(d(W), T)),
    ("embedding_grad", lambda d: F.embedding_grad(d(X), T, 5)),
    ("embedding_grad", lambda d: F.embedding_grad(X, T, 5, out=d(W), accumulate=True)),
])
def test_tangents_are_refused(name, call, grad):
    """A dual argument would give a result without its tangent."""
    fw = torch.autograd.forward_ad
    with fw.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError, match=name):
            call(lambda x: fw.make_dual(x, torch.ones_like(x)))
    with pytest.raises(NotImplementedError, match=name):
        def f(x):
            return call(lambda like: x[:like.numel()].view(like.shape))
        torch.func.jvp(f, (torch.zeros(40),), (torch.ones(40),))


def test_lookup_takes():
    assert F.lookup_takes(W) and F.lookup_takes(W.t()) and F.lookup_takes(W.half())
    for x in (W.double(), W[0], W[:0], W[:, :0], torch.zeros(2, 65537),
              torch.zeros(1, 1).expand(1 << 30, 1), W.clone().requires_grad_()):
        assert not F.lookup_takes(x)
    with torch.no_grad():
        assert F.lookup_takes(W.clone().requires_grad_())
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        assert not F.lookup_takes(fw.make_dual(W, W))


class C:
    """One entry's arguments by name, valid ones for pointers that are never read."""
    XENT = dict(type=1, X=256, sxn=8, sxd=1, W=256, swv=8, swd=1, bias=None, targets=256,
                ignore=-100, N=4, V=5, D=8)
    FWD = dict(XENT, loss=256, logZ=256, reduction=0, reduced=None, count=None, ws=256, nws=1 << 40,
               stream=None)
    BWD = dict(XENT, logZ=256, dloss=256, ds=1, count=None, dlogZ=None, dX=256, dW=256, dbias=None,
               ws=256, nws=1 << 40, stream=None)
    EFWD = dict(type=1, table=256, tsv=8, tsd=1, ids=256, ignore=-100, N=4, V=5, D=8, scale=1.0,
                out=256, stream=None)
    EBWD = dict(type=1, dout=256, dsn=8, dsd=1, ids=256, ignore=-100, N=4, V=5, D=8, scale=1.0,
                dtable=256, ws=256, nws=1 << 40, flags=0, stream=None)


@pytest.mark.parametrize("entry,args,change,code,match", [
    (e, a, ch, code, m)
    for e, a in (("fgmm_xent_fwd", C.FWD), ("fgmm_xent_bwd", C.BWD),
                 ("fgmm_embed_fwd", C.EFWD), ("fgmm_embed_bwd", C.EBWD))
    for ch, code, m in (
        (dict(type=3), 1, "unknown type"), (dict(N=-1), 1, "invalid shape"),
        (dict(V=0), 1, "invalid shape"), (dict(D=0), 1, "invalid shape"),
        (dict(N=1 << 30), 3, "exceeds"), (dict(V=1 << 30), 3, "exceeds"),
        (dict(D=65537), 3, "exceeds"))
] + [
    ("fgmm_xent_fwd", C.FWD, dict(X=None), 1, "null pointer"),
    ("fgmm_xent_fwd", C.FWD, dict(W=None), 1, "null pointer"),
    ("fgmm_xent_fwd", C.FWD, dict(targets=None), 1, "null pointer"),
    ("fgmm_xent_fwd", C.FWD, dict(loss=None), 1, "null pointer"),
    ("fgmm_xent_fwd", C.FWD, dict(reduction=2), 1, "null pointer"),
    ("fgmm_xent_fwd", C.FWD, dict(reduction=3), 1, "unknown reduction"),
    ("fgmm_xent_fwd", C.FWD, dict(sxn=-8), 1, "negative stride"),
    ("fgmm_xent_fwd", C.FWD, dict(W=257), 1, "not aligned"),
    ("fgmm_xent_fwd", C.FWD, dict(bias=258), 1, "not aligned"),
    ("fgmm_xent_bwd", C.BWD, dict(ds=2), 1, "dloss_stride"),
    ("fgmm_xent_bwd", C.BWD, dict(logZ=None), 1, "null pointer"),
    ("fgmm_xent_bwd", C.BWD, dict(dX=257), 1, "not aligned"),
    ("fgmm_xent_bwd", C.BWD, dict(N=(1 << 30) - 1, V=(1 << 30) - 1), 3, "split the rows"),
    ("fgmm_embed_fwd", C.EFWD, dict(out=None), 1, "null pointer"),
    ("fgmm_embed_fwd", C.EFWD, dict(tsd=-1), 1, "negative stride"),
    ("fgmm_embed_bwd", C.EBWD, dict(dtable=None), 1, "null pointer"),
    ("fgmm_embed_bwd", C.EBWD, dict(flags=2), 1, "unknown flags"),
    ("fgmm_embed_bwd", C.EBWD, dict(dout=257), 1, "not aligned"),
])
def test_c_entries_refuse_before_any_device_call(lib, entry, args, change, code, match):
    got = getattr(lib, entry)(*dict(args, **change).values())
    assert got == code, lib.fgmm_last_error()
    message = lib.fgmm_last_error().decode()
    assert match in message and entry in message


@pytest.mark.parametrize("change", [
    dict(dout=4096, dtable=4096),                              # the gradient over its own input
    dict(dout=1 << 20, dtable=(1 << 20) - 16),                 # its last row reaches into dout
    dict(dtable=1 << 20, dout=(1 << 20) + 16, dsn=0),          # one row for all positions, inside
    dict(dtable=1 << 20, ids=(1 << 20) + 8, dout=1 << 24),
    dict(dtable=1 << 40, dout=1 << 20, dsn=1 << 38),           # rows far apart reach over it
])
def test_embed_bwd_refuses_overlapping_arrays(lib, change):
    assert set(change) <= set(C.EBWD)
    assert lib.fgmm_embed_bwd(*dict(C.EBWD, **change).values()) == 1
    message = lib.fgmm_last_error().decode()
    assert "overlaps" in message and "fgmm_embed_bwd" in message


def test_workspace_sizes(lib):
    for back in (0, 1):
        for kind in (0, 1, 2):
            sizes = [lib.fgmm_xent_workspace_bytes(back, kind, n, 5000, 256, 1024, 256, 1, 0)
                     for n in (0, 1, 2, 1000)]
            assert sizes == sorted(sizes) and sizes[1] > 0
            for at, s0, s1 in ((1026, 256, 1), (1024, 257, 1), (1024, 1, 5000), (1024, 0, 1)):
                one, two = (lib.fgmm_xent_workspace_bytes(back, kind, n, 5000, 256, at, s0, s1, 0)
                            for n in (1, 2))
                # one row reads W in place; two 16-bit rows have it copied, two fp32 rows not
                assert one < 2 * 5000 * 255
                assert (two > sizes[2] + 2 * 5000 * 255) == (kind != 0)
    assert lib.fgmm_xent_workspace_bytes(0, 9, 10, 10, 10, 1024, 16, 1, 0) == 0
    assert lib.fgmm_embed_workspace_bytes(1000, 50, 8) > 0
    assert lib.fgmm_embed_workspace_bytes(-1, 50, 8) == 0


@pytest.mark.parametrize("kind", [0, 1, 2], ids=["fp32", "bf16", "fp16"])
def test_xent_bwd_counts_dbias_without_a_bias(lib, kind):
    """bias may be NULL where dbias is asked: its parts need their place in the workspace."""
    N, V, D = 5000, 3000, 64
    args = dict(C.BWD, type=kind, N=N, V=V, D=D, swv=D, sxn=D, dbias=256)
    without = lib.fgmm_xent_workspace_bytes(1, kind, N, V, D, 256, D, 1, 0)
    with_parts = lib.fgmm_xent_workspace_bytes(1, kind, N, V, D, 256, D, 1, 1)
    assert with_parts > without
    for bias in (None, 256):
        got = lib.fgmm_xent_bwd(*dict(args, bias=bias, nws=without).values())
        assert got == 2, (bias, got, lib.fgmm_last_error())
        assert str(with_parts) in lib.fgmm_last_error().decode()


@pytest.mark.parametrize("kind", [0, 1, 2], ids=["fp32", "bf16", "fp16"])
def test_bias_workspace_does_not_grow_with_the_rows(lib, kind):
    def extra(N, V, D=64):
        return [lib.fgmm_xent_workspace_bytes(1, kind, N, V, D, 256, D, 1, b) for b in (0, 1)]
    for V in (1000, 5000, 131072):
        without, given = extra(1 << 17, V)
        # five chunks of a piece's 32 MB of words: at most this share of them a part
        assert given - without <= 4 * V * (5 * 32 * 2 ** 20 / (128 * 2 * min(V, 4096)) + 256) + 4096
        more, much_more = extra(1 << 22, V)
        assert abs((much_more - more) - (given - without)) <= 4096 or V == 1000
    without, given = extra(1 << 22, 1000)
    assert extra(1 << 26, 1000)[1] - extra(1 << 26, 1000)[0] == given - without


@pytest.mark.parametrize("kind", [0, 1, 2], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("D", [1, 64, 128, 129, 1000, 1024, 1025, 4096, 8192, 16384, 65536])
def test_xent_bwd_takes_the_stated_sizes(lib, D, kind):
    """N V up to 2^55 / max(D, 1024) is not refused for its size (no workspace is given, which
    is found before anything runs)."""
    for log_v in range(8, 30, 3):
        V = (1 << log_v) - 1
        N = min((1 << 30) - 1, (1 << 55) // max(D, 1024) // V)
        got = lib.fgmm_xent_bwd(*dict(C.BWD, type=kind, N=N, V=V, D=D, swv=D, sxn=D, nws=0).values())
        assert got == 2, (N, V, lib.fgmm_last_error())


def test_no_unbounded_barrier_between_the_roles():
    """The persistent kernel's warps leave one by one after a wait that gave up, so that they
    may meet at mbarriers with bounded waits only: a hardware barrier of some of a block's
    warps would keep the others for good."""
    path = os.path.join(os.path.dirname(L.__file__), "csrc", "fgmm_xent_mma.cuh")
    source = open(path).read()
    assert "bar.sync" not in source and "barrier.sync" not in source
    body = source[source.index("xent_mma_kernel("):]
    roles = body[body.index("regs_down<72>"):body.rindex("tc_fence_before();")]
    assert "__syncthreads" not in roles and "cluster_sync_all" not in roles


def test_oracle_against_autograd():
    """The plain form the GPU tests compare with, against torch's own gradients in 64 bits."""
    X, W, t, c = R.problem(40, 30, 12, torch.float32, ignored=0.3, bias=True, device="cpu")
    w, z = torch.rand(40), torch.rand(40)
    ref = R.xent(X, W, t, c, w=w, dlogZ=z)
    X, W, c = (x.double().requires_grad_() for x in (X, W, c))
    S = X @ W.t() + c
    loss = torch.nn.functional.cross_entropy(S, t, reduction="none", ignore_index=R.IGNORE)
    keep = (t != R.IGNORE).double()
    ((loss * w).sum() + (torch.logsumexp(S, 1) * z * keep).sum()).backward()
    for got, name in ((loss.detach(), "loss"), (X.grad, "dX"), (W.grad, "dW"), (c.grad, "dbias")):
        assert float((got - ref[name]).abs().max()) < 1e-12
    g, ids = torch.randn(40, 6), torch.randint(0, 9, (40,))
    e = torch.zeros(9, 6, dtype=torch.float64, requires_grad=True)
    (e[ids] * 0.3 * g.double()).sum().backward()
    assert float((R.embed_grad(g, ids, 9, 0.3)[0] - e.grad).abs().max()) < 1e-12
