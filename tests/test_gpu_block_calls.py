"""GPU (-m gpu): calls of the trainable block's operators (layer_norm, linear_act, GradClip / clip_grad_norm_) next to the ordinary ones:
values that are not finite, tensors that stand for their memory in another way, operands that change between the passes."""
import pytest
import torch

import hopmi

pytestmark = pytest.mark.gpu
ops = hopmi.ops
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _dev():
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    return torch.device("cuda:0")


def _rng(seed):
    return torch.Generator(device=_dev()).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=_dev())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("M,K,N", [(8, 16, 24), (100, 40, 21), (300, 72, 64)])
def test_relu_drops_what_arrives_at_inactive_units(M, K, N, dtype):
    """dz = where(z > 0, dy, 0): an infinity or a NaN of dy at an inactive unit changes nothing, at an active one it stays in its row of
    dx, its row of dw and its bias gradient."""
    t = TYPES[dtype]
    g = _rng(M + N)
    leaves = [v.to(t).requires_grad_() for v in (_randn(g, M, K), _randn(g, N, K), _randn(g, N))]
    y = ops.linear_act(*leaves, activation="relu")
    dy = _randn(g, M, N).to(t)
    off = y.detach() == 0
    plain = torch.where(off, torch.zeros_like(dy), dy)
    want = torch.autograd.grad(y, leaves, plain, retain_graph=True)
    bad = dy.clone()
    k = off.flatten().nonzero()[:, 0]
    for i, v in enumerate((float("inf"), float("-inf"), float("nan"))):
        bad.view(-1)[k[i::3]] = v
    got = torch.autograd.grad(y, leaves, bad, retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    row, col = (~off).nonzero()[0].tolist()
    bad[row, col] = float("inf")
    dx, dw, db = torch.autograd.grad(y, leaves, bad)
    assert not dx[row].isfinite().any() and not dw[col].isfinite().any() and db[col] == float("inf")
    rows, cols = torch.arange(M, device=_dev()) != row, torch.arange(N, device=_dev()) != col
    assert torch.equal(dx[rows], want[0][rows]) and torch.equal(dw[cols], want[1][cols]) and torch.equal(db[cols], want[2][cols])
    # a NaN before the activation is not above zero either
    b = leaves[2].detach().clone()
    b[0] = float("nan")
    b.requires_grad_()
    y = ops.linear_act(leaves[0], leaves[1], b, activation="relu")
    gb = torch.autograd.grad(y, b, dy)[0]
    assert y[:, 0].isnan().all() and gb[0] == 0


@pytest.mark.parametrize("M,N", [(8, 16), (150, 24), (90, 1), (1, 40)])
def test_a_gradient_with_a_pending_negation(M, N):
    """autograd hands a backward pass views whose sign is still to be applied (the imaginary part of a conjugate): dense ones, ones with a
    single column, strided ones."""
    g = _rng(M)
    dy = _randn(g, M, N)
    wide = _randn(g, M, 2 * N)
    forms = [(torch._neg_view(-dy), dy), (torch._neg_view(wide[:, :N]), -wide[:, :N]), (torch._neg_view(wide[:, ::2]), -wide[:, ::2]),
             (torch.complex(dy, dy).conj().imag, -dy)]
    x, w, b = (_randn(g, *s).requires_grad_() for s in ((M, N), (N,), (N,)))
    for neg, plain in forms:
        assert neg.is_neg() and not plain.is_neg()
        a, c = (torch.autograd.grad(ops.layer_norm(x, w, b), [x, w, b], d) for d in (neg, plain))
        assert all(torch.equal(p, q) for p, q in zip(a, c))
    for act in ("none", "gelu"):
        for need in ((True, True, True), (False, False, True)):
            leaves = [_randn(g, *s).bfloat16().requires_grad_(n) for s, n in zip(((M, 40), (N, 40), (N,)), need)]
            wanted = [v for v in leaves if v.requires_grad]
            for neg, plain in [(torch._neg_view(-dy.bfloat16()), dy.bfloat16()), (torch._neg_view(wide.bfloat16()[:, :N]), -wide.bfloat16()[:, :N])]:
                a, c = (torch.autograd.grad(ops.linear_act(*leaves, activation=act), wanted, d) for d in (neg, plain))
                assert all(torch.equal(p, q) for p, q in zip(a, c))
    # as it comes about: through the imaginary part of a conjugate
    y = ops.layer_norm(x, w, b)
    got = torch.autograd.grad((torch.complex(y, 2 * y).conj().imag * dy).sum(), x)[0]
    assert torch.equal(got, torch.autograd.grad(ops.layer_norm(x, w, b), x, -2 * dy)[0])


def test_recorded_step_follows_a_changed_limit(monkeypatch):
    """args.max_grad_norm may change between calls of a recorded step: the call with the new limit clips by it, and the step is recorded
    again (it does not stay eager)."""
    from oracle.golden_util import step_args
    from test_gpu_graph import _deterministic_draws, _pair
    _deterministic_draws(monkeypatch)
    m, d, inp = _pair(9, _dev())
    batch = (inp["in_audio"], inp["log_melspec"], inp["text"], inp["target_dir_vec"], inp["vid_indices"])
    g = torch.optim.Adam([p for p in m.parameters() if p.requires_grad], lr=1e-4, betas=(0.5, 0.999))
    o = torch.optim.Adam(d.parameters(), lr=1e-4, betas=(0.5, 0.999))
    args = step_args(9)
    run = hopmi.GraphedTrainStep(args, m, d, g, o, eager_calls=1)

    def call():
        run(0, *batch)
        torch.cuda.synchronize()
        return sum(float(p.grad.double().square().sum()) for p in m.parameters() if p.grad is not None) ** 0.5

    free = [call() for _ in range(3)]
    assert (run.n_eager, run.n_replay) == (1, 2)
    for limit, eager, replay in ((0.125 * free[-1], 2, 4), (0.25 * free[-1], 3, 6)):
        args.max_grad_norm = limit
        # far below the norm of every step here, so the gradients a step leaves behind have it as theirs: 1e-6 in the formula's
        # denominator, one rounding per value
        norms = [call() for _ in range(3)]
        assert all(abs(n - limit) <= 1e-5 * free[-1] for n in norms), (norms, limit)
        assert (run.n_eager, run.n_replay) == (eager, replay)
    args.max_grad_norm = None
    assert all(call() > 0.5 * free[-1] for _ in range(3)) and (run.n_eager, run.n_replay) == (4, 8)


def test_grad_clip_of_lazy_copies():
    """A tensor that shares its memory with another until one of them is written: clipping in place writes it, so the other keeps its
    values; read only (out given), it may go on sharing."""
    base = torch.full((1000,), 2.0, device=_dev())
    a, b = torch._lazy_clone(base), torch._lazy_clone(base)
    plan = ops.GradClip([a, b])
    norm = plan.clip_(1.0)
    want = (2000 * 4) ** 0.5
    assert abs(float(norm) - want) <= 2 * 2.0 ** -24 * want
    assert (base == 2).all() and all(torch.allclose(t, torch.full_like(t, 2 / want), rtol=1e-6) for t in (a, b))
    c, o = torch._lazy_clone(base), torch.zeros(1000, device=_dev())
    ops.GradClip([c], out=[o]).clip_(1.0)
    assert (base == 2).all() and (c == 2).all() and torch._C._is_cow_tensor(c) and (o < 1).all()
    d = torch._lazy_clone(base)                                                  # written through a lazy output: only that one
    ops.GradClip([torch.ones(1000, device=_dev())], out=[d]).clip_(1.0)
    assert (base == 2).all() and (d < 1).all()


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_a_second_derivative_is_refused_for_every_operand(act):
    """linear_act's first gradients depend on the bias through act'(z): that way too leads to the error, not to a missing gradient."""
    g = _rng(4)
    x, w, b, r = (_randn(g, *s).bfloat16().requires_grad_() for s in ((80, 16), (24, 16), (24,), (80, 24)))
    gx, gw, gb = torch.autograd.grad(ops.linear_act(x, w, b, r, act).sum(), [x, w, b], create_graph=True)
    for first in (gx, gw, gb):
        for leaf in [x, w] + [b] * (act != "none"):
            with pytest.raises(RuntimeError, match="differentiable once"):
                torch.autograd.grad(first.float().sum(), leaf, allow_unused=True, retain_graph=True)
        # neither the residual nor, without an activation, the bias is in them
        assert torch.autograd.grad(first.float().sum(), [r] + [b] * (act == "none"), allow_unused=True, retain_graph=True)[0] is None
    # only the bias is trained: its gradient is made of it all the same
    gb = torch.autograd.grad(ops.linear_act(x.detach(), w.detach(), b, activation="gelu").sum(), b, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(gb.float().sum(), b)
    # the incoming gradient
    dy = torch.ones(80, 24, device=_dev(), dtype=torch.bfloat16).requires_grad_()
    gx = torch.autograd.grad(ops.linear_act(x, w, b, r, act), x, dy, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(gx.float().sum(), dy)
    # layer norm: each of its operands
    lx, lw, lb = (_randn(g, *s).requires_grad_() for s in ((80, 16), (16,), (16,)))
    for ww, bb in ((lw, lb), (lw, None), (None, lb), (None, None)):
        leaves = [t for t in (lx, ww, bb) if t is not None]
        for first in torch.autograd.grad(ops.layer_norm(lx, ww, bb).square().sum(), leaves, create_graph=True):
            for leaf in leaves:
                with pytest.raises(RuntimeError, match="differentiable once"):
                    torch.autograd.grad(first.sum(), leaf, retain_graph=True)


@pytest.mark.parametrize("M,K,N", [(40, 64, 48), (150, 64, 48), (150, 61, 45)])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_an_operand_may_change_where_no_wanted_gradient_reads_it(M, K, N, act):
    """dx reads w, dw reads x, db neither; layer norm's dx reads x and weight, dweight x, dbias none.  What is not read is not kept: it may
    be overwritten between the passes (a frozen layer's input by the next in-place operation), and what is read is still watched."""
    g = _rng(M + K)
    t = torch.bfloat16
    x, w, b = _randn(g, M, K).to(t), (_randn(g, N, K) / 8).to(t), _randn(g, N).to(t)
    dy = _randn(g, M, N).to(t)
    reads = {0: {1}, 1: {0}, 2: set()}
    for i in range(3):
        leaves = [v.clone().requires_grad_(i == k) for k, v in enumerate((x, w, b))]
        want = torch.autograd.grad(ops.linear_act(*leaves, activation=act), leaves[i], dy)[0]
        for j in range(3):
            leaves = [v.clone().requires_grad_(i == k) for k, v in enumerate((x, w, b))]
            given = [v * 1 for v in leaves]
            y = ops.linear_act(*given, activation=act)
            with torch.no_grad():
                given[j].add_(1)
            if j in reads[i] and K % 8 == 0:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    torch.autograd.grad(y, leaves[i], dy)
            else:                                                                # (rows copied for the product are the product's own)
                if j in reads[i] and M <= 64:
                    continue
                assert torch.equal(torch.autograd.grad(y, leaves[i], dy)[0], want), (i, j)
    x, w, b = (_randn(g, *s) for s in ((M, K), (K,), (K,)))
    dy = _randn(g, M, K)
    reads = {0: {0, 1}, 1: {0}, 2: set()}
    for i in range(3):
        leaves = [v.clone().requires_grad_(i == k) for k, v in enumerate((x, w, b))]
        want = torch.autograd.grad(ops.layer_norm(*leaves), leaves[i], dy)[0]
        for j in range(3):
            leaves = [v.clone().requires_grad_(i == k) for k, v in enumerate((x, w, b))]
            given = [v * 1 for v in leaves]
            y = ops.layer_norm(*given)
            with torch.no_grad():
                given[j].add_(1)
            if j in reads[i]:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    torch.autograd.grad(y, leaves[i], dy)
            else:
                assert torch.equal(torch.autograd.grad(y, leaves[i], dy)[0], want), (i, j)


def test_frozen_weights_do_not_keep_the_input():
    """With w frozen, x is not held by the tape: its memory is free again when the caller lets go of it."""
    t = torch.bfloat16
    w = torch.zeros(64, 4096, device=_dev(), dtype=t)
    leaf = torch.zeros(4096, 4096, device=_dev(), dtype=t).requires_grad_()
    x = leaf * 1                                                                 # 32 MiB
    y = ops.linear_act(x, w)
    held = torch.cuda.memory_allocated()
    del x
    assert held - torch.cuda.memory_allocated() >= 32 << 20
    assert torch.autograd.grad(y.sum(), leaf)[0].shape == leaf.shape


@pytest.mark.parametrize("M", [40, 150])
def test_operands_are_copied_once(M):
    """A transposed weight, or rows without a common stride, are made dense once, in the forward pass, and the backward pass takes that
    copy: allocations counted per call."""
    def count(f):
        n = torch.cuda.memory_stats()["allocation.all.allocated"]
        r = f()
        return r, torch.cuda.memory_stats()["allocation.all.allocated"] - n

    g = _rng(M)
    t = torch.bfloat16
    w = (_randn(g, 64, 48).to(t) / 8).t().requires_grad_()                       # (48, 64), contiguous along its rows' number
    x = _randn(g, 2, M, 64).to(t)[:, :M // 2].transpose(0, 1).requires_grad_()   # rows of two blocks, interleaved: no common stride
    wd, xd = w.detach().contiguous().requires_grad_(), x.detach().contiguous().requires_grad_()
    dy = _randn(g, M // 2, 2, 48).to(t)
    y0, forward = count(lambda: ops.linear_act(xd, wd))
    want, backward = count(lambda: torch.autograd.grad(y0, [xd, wd], dy))
    for xx, ww, copies in ((x, wd, 1), (xd, w, 1), (x, w, 2)):
        y, n = count(lambda: ops.linear_act(xx, ww))
        assert n == forward + copies and torch.equal(y, y0)
        got, n = count(lambda: torch.autograd.grad(y, [xx, ww], dy))
        assert n == backward and all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("M,K,N", [(40, 64, 48), (150, 61, 45)])
def test_saved_tensors_that_travel_and_recomputed_blocks(M, K, N):
    """What the operators keep may be packed away and come back as another tensor (dense, elsewhere), and a block may be run again
    in its backward pass."""
    from torch.utils.checkpoint import checkpoint
    g = _rng(M)
    t = torch.bfloat16
    x = _randn(g, M, 2 * K).to(t)[:, ::2].requires_grad_()
    w, b = (_randn(g, N, K) / 8).to(t).requires_grad_(), _randn(g, N).to(t).requires_grad_()
    lw, lb = _randn(g, N).requires_grad_(), _randn(g, N).requires_grad_()
    dy = _randn(g, M, N).to(t)
    leaves = [x, w, b, lw, lb]
    block = lambda *v: ops.layer_norm(ops.linear_act(*v[:3], activation="gelu"), v[3], v[4])
    want = torch.autograd.grad(block(*leaves), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = block(*leaves)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, dy), want))
    y = checkpoint(block, *leaves, use_reentrant=False)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, dy), want))


def test_calls_from_several_threads():
    """Forward and backward passes from several Python threads at once, each on a stream of its own."""
    import threading
    g = _rng(8)
    t = torch.bfloat16
    sets = []
    for k in range(3):
        v = [_randn(g, 150 + k, 72).to(t), (_randn(g, 56, 72) / 8).to(t), _randn(g, 56).to(t), _randn(g, 56), _randn(g, 56), _randn(g, 150 + k, 56).to(t)]

        def run(v=v):
            leaves = [a.clone().requires_grad_() for a in v[:5]]
            y = ops.layer_norm(ops.linear_act(*leaves[:3], activation="silu"), *leaves[3:])
            grads = torch.autograd.grad(y, leaves, v[5])
            out = [torch.empty(a.shape, device=a.device) for a in grads]
            return [y.detach(), *grads, ops.GradClip(grads, out=out).clip_(0.5), *out]

        sets.append((run, run()))
    torch.cuda.synchronize()
    bad = []

    def work(run, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [run() for _ in range(10)]
            torch.cuda.current_stream().synchronize()
        if not all(torch.equal(p, q) for r in got for p, q in zip(r, want)):
            bad.append(run)

    threads = [threading.Thread(target=work, args=s) for s in sets]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad


@pytest.mark.parametrize("M,N,shape", [(16384, 64, (64,)), (4352, 768, (768,)), (4352, 768, (4352, 1)), (4352, 768, (1,)), (64, 16384, (64, 1))])
def test_a_broadcast_residual_in_a_recorded_backward(M, N, shape):
    """The residual's gradient is then a sum by torch, which may record more than kernels: every replay against the eager result, with eager
    work between them."""
    g = _rng(M + N)
    t = torch.bfloat16
    x, w, r = _randn(g, M, 64).to(t), (_randn(g, N, 64) / 8).to(t), _randn(g, *shape).to(t).requires_grad_()
    dy = _randn(g, M, N).to(t)
    f = lambda: torch.autograd.grad(ops.linear_act(x, w, None, r), r, dy)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = f()
    for _ in range(6):
        dy.copy_(_randn(g, M, N))
        want = f().clone()
        (_randn(g, 1000, 1000) @ _randn(g, 1000, 1000)).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# (shape of x w^T, shape of the residual): each pattern of repeated axes, few and many of them, columns above and below a wave's width
BROADCAST = [((150, 48), (48,)), ((150, 48), (1, 48)), ((150, 48), (150, 1)), ((150, 48), (1,)), ((150, 48), (1, 1)), ((4352, 768), (768,)),
             ((4352, 768), (4352, 1)), ((4352, 768), (1,)), ((9, 17, 70), (17, 70)), ((9, 17, 70), (9, 1, 70)), ((9, 17, 70), (9, 17, 1)),
             ((9, 17, 70), (1, 17, 1)), ((9, 17, 70), (9, 1, 1)), ((3, 5, 7, 33), (5, 1, 33)), ((3, 5, 7, 33), (3, 1, 7, 1)),
             ((200, 1, 24), (24,)), ((1, 40), (40,)), ((20001, 3), (3,)), ((20001, 3), (20001, 1)), ((2, 3000, 130), (2, 1, 130)),
             ((70000, 8), (70000, 1)), ((2100, 63), (63,)), ((2100, 64), (64,)), ((2100, 65), (65,)), ((0, 8), (8,)), ((5, 0, 8), (5, 1, 8)),
             ((1025, 1000), (1,))]


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape,rshape", BROADCAST)
def test_gradient_of_a_broadcast_residual(shape, rshape, t):
    g = _rng(sum(shape) + len(rshape))
    K = 16
    x, w = _randn(g, *shape[:-1], K).to(t), (_randn(g, shape[-1], K) / 4).to(t)
    r = _randn(g, *rshape).to(t).requires_grad_()
    dy = (_randn(g, *shape) + 0.1).to(t)
    y = ops.linear_act(x, w, None, r, "gelu")
    assert torch.equal(y, ops.linear_act(x, w, None, r.detach().expand(shape).contiguous(), "gelu"))
    wide = torch.full((*shape[:-1], shape[-1] + 5), 7.0, device=_dev(), dtype=t)
    wide[..., 2:2 + shape[-1]] = dy
    want = dy.double().sum_to_size(rshape)
    mags = dy.double().abs().sum_to_size(rshape)
    n = dy.numel() // max(1, r.numel())
    for d in (dy, wide[..., 2:2 + shape[-1]]):
        got = torch.autograd.grad(y, r, d, retain_graph=True)[0]
        assert got.dtype == t and got.shape == r.shape
        if n == 0:
            assert not got.any()
            continue
        # half a step of the type, and at most one rounding of 2^-24 of the magnitudes per addition
        tol = torch.finfo(t).eps / 2 * want.abs() + n * 2.0 ** -24 * mags + torch.finfo(t).tiny * torch.finfo(t).eps
        # (a sum that rounds past the type's largest value is an infinity: 4352 x 768 values of mean 0.1 add to 334 000, fp16 ends at 65 520)
        over = want.abs() >= torch.finfo(t).max * (1 + torch.finfo(t).eps / 4)
        assert (got.double()[over] == want.sign()[over] * float("inf")).all()
        assert ((got.double() - want).abs() <= tol)[~over].all(), float(((got.double() - want).abs() - tol)[~over].max())
        assert torch.equal(got, torch.autograd.grad(y, r, d, retain_graph=True)[0])          # the same bits every time


def test_axis_sum_writes_nothing_else():
    """Sums next to other values, of a large and a small axis in both forms, and of a long one that is cut into groups."""
    from hopmi import _lib
    L = _lib.lib()
    st = torch.cuda.current_stream().cuda_stream
    g = _rng(77)
    for outer, R, inner in ((1, 4352, 768), (3, 70, 65), (1, 100003, 1), (5, 9, 63), (4099, 12, 3), (1, 1, 1), (2, 50000, 64), (70000, 2, 7),
                            (70000, 8, 8), (2100, 9, 8), (2100, 5000, 1), (2100, 130, 33), (30, 1, 50), (300000, 3, 2)):
        for it, ot in ((0, 0), (1, 0), (1, 1), (0, 2)):
            v = _randn(g, outer, R, inner).to({0: torch.float32, 1: torch.bfloat16}[it])
            to = {0: torch.float32, 1: torch.bfloat16, 2: torch.float16}[ot]
            buf = torch.full((outer * inner + 16,), 7.0, device=_dev(), dtype=to)
            n = L.hopmi_axis_sum_ws_floats(outer, R, inner)
            ws = torch.full((n + 8,), 5.0, device=_dev())
            assert L.hopmi_axis_sum(v.data_ptr(), it, buf[8:].data_ptr(), ot, outer, R, inner, ws.data_ptr() if n else None, st) == 0
            got, want = buf[8:-8].double().view(outer, inner), v.double().sum(1)
            tol = torch.finfo(to).eps / 2 * want.abs() + R * 2.0 ** -24 * v.double().abs().sum(1)
            assert ((got - want).abs() <= tol).all() and (buf[:8] == 7).all() and (buf[-8:] == 7).all() and (ws[n:] == 5).all()
