"""GPU (-m gpu): every form that linear_act's products take, and the loops over rows of layer norm's kernels, against 64-bit results.

Tolerances are counted as in test_gpu_block.py: half a step of the output's type, plus the roundings of 32-bit arithmetic on the way."""
import pytest
import torch

import hopmi
import linear_forms as lf
from test_gpu_block import U32, _check_linear, _dev, _half_step, _randn, _rng, _tiny, check

pytestmark = pytest.mark.gpu
ops = hopmi.ops
TYPES = [torch.bfloat16, torch.float16]


def _cases(sizes):
    return [pytest.param(*size, TYPES[i % 2], id="-".join(map(str, (*key, *size))) if isinstance(key, tuple) else f"{key}-{size}")
            for i, (key, size) in enumerate(sizes.items())]


@pytest.mark.parametrize("M,K,N,t", _cases(lf.ALONE["y"]) + _cases(lf.FEW))
def test_forward_forms(M, K, N, t):
    _check_linear(M, K, N, t, "gelu", True, True, False)


@pytest.mark.parametrize("M,K,N,t", _cases(lf.ALONE["dx"]))
def test_input_gradient_alone(M, K, N, t):
    """A frozen weight: dx = dz w in a launch of its own (and the join of its split)."""
    g = _rng(M + K)
    x, w, dy = _randn(g, M, K).to(t).requires_grad_(), (_randn(g, N, K) * K ** -0.5).to(t), _randn(g, M, N).to(t)
    got = torch.autograd.grad(ops.linear_act(x, w), x, dy)[0]
    assert torch.equal(got, torch.autograd.grad(ops.linear_act(x, w), x, dy)[0])
    D, W = dy.double(), w.double()
    want = D @ W
    check(got, want, _half_step(t) * want.abs() + (N + 2) * 2 * U32 * (D.abs() @ W.abs()) + _tiny(t), "dx")


@pytest.mark.parametrize("M,K,N,t", _cases(lf.ALONE["dw"]))
def test_weight_gradient_alone(M, K, N, t):
    """An input that takes no gradient: dw = dz^T x in a launch of its own."""
    g = _rng(M + N)
    x, w, dy = _randn(g, M, K).to(t), (_randn(g, N, K) * K ** -0.5).to(t).requires_grad_(), _randn(g, M, N).to(t)
    got = torch.autograd.grad(ops.linear_act(x, w), w, dy)[0]
    assert torch.equal(got, torch.autograd.grad(ops.linear_act(x, w), w, dy)[0])
    D, X = dy.double(), x.double()
    want = D.t() @ X
    check(got, want, _half_step(t) * want.abs() + (M + 2) * 2 * U32 * (D.abs().t() @ X.abs()) + _tiny(t), "dw")


@pytest.mark.parametrize("M,K,N,t", _cases(lf.PAIRED) + _cases(lf.SEPARATE))
def test_both_gradients(M, K, N, t):
    _check_linear(M, K, N, t, "silu", True, False, True)


# ------------------------------------------------------------------------------------------------------- layer norm's row loops
# (rows, width in vectors of 16 bytes, elements behind the last one): more rows than the grids have places for, and no multiple of them --
# backward: 4096 rows up to 128 vectors, 2048 up to 256 (a wave to a row), 512 up to 512 / 1024 / 2048 (256 / 512 / 1024 threads), 512 and, for
# its column sums, 256 beyond; forward: 8192, 1536, 1024, 512, 512
LN_ROWS = [(9001, 4, 1), (4352, 96, 0), (8301, 128, 3), (8203, 129, 0), (2101, 255, 3), (1601, 257, 1), (1537, 512, 0), (1101, 1000, 2), (1027, 1024, 0),
           (601, 2048, 0), (1101, 2047, 3), (601, 2049, 1), (300, 2500, 2)]


@pytest.mark.parametrize("t,wt", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)],
                         ids=["fp32", "bf16", "fp16-fp32"])
@pytest.mark.parametrize("M,vecs,tail", LN_ROWS)
def test_layer_norm_row_loops(M, vecs, tail, t, wt):
    D = vecs * (16 // t.itemsize) + tail
    g = _rng(M + D)
    buf = torch.zeros(M, D + (M % 3) * 5, device=_dev(), dtype=t)
    buf[:, :D] = _randn(g, M, D) * torch.exp(0.3 * _randn(g, M, 1)) + 0.7
    x = buf[:, :D].requires_grad_()
    w, b = (1 + 0.2 * _randn(g, D)).to(wt).requires_grad_(), (0.2 * _randn(g, D)).to(wt).requires_grad_()
    dy = _randn(g, M, D).to(t)
    y = ops.layer_norm(x, w, b, 1e-5)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    again = torch.autograd.grad(ops.layer_norm(x, w, b, 1e-5), [x, w, b], dy)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, dw, db)))           # the same bits every time
    X, W, B, G = x.detach().double(), w.detach().double(), b.detach().double(), dy.double()
    mu = X.mean(-1, keepdim=True)
    r = 1 / ((X - mu).square().mean(-1, keepdim=True) + 1e-5).sqrt()
    xh = (X - mu) * r
    # roundings of a row's sum: a thread's own additions (four vectors of eight and one value, or D / 1024), ten levels across threads, a
    # dozen around them
    n = 55 + D / 1024
    exh = n * U32 * ((X.abs().mean(-1, keepdim=True) + X.abs()) * r + 2 * xh.abs())
    want = xh * W + B
    check(y, want, _half_step(t) * want.abs() + exh * W.abs() + 2 * U32 * ((xh * W).abs() + B.abs()) + _tiny(t), "y")
    gw = G * W
    m0, m1 = gw.mean(-1, keepdim=True), (gw * xh).mean(-1, keepdim=True)
    want = r * (gw - m0 - xh * m1)
    em0 = n * U32 * gw.abs().mean(-1, keepdim=True)
    em1 = n * U32 * (gw * xh).abs().mean(-1, keepdim=True) + (gw.abs() * exh).mean(-1, keepdim=True)
    tol = r * (4 * U32 * gw.abs() + em0 + xh.abs() * em1 + exh * m1.abs() + 4 * U32 * (m0.abs() + (xh * m1).abs())) + n * U32 * want.abs()
    check(dx, want, _half_step(t) * want.abs() + tol + _tiny(t), "dx")
    # roundings of a column's sum: the rows of a wave or workgroup one after the other (at least 256 of them side by side), the four waves,
    # the partial rows of up to 1024 workgroups by sixteen waves, these sixteen, and the products' own
    ns = M / 256 + 1 + 4 + 1024 / 16 + 16 + 4
    want = (G * xh).sum(0)
    check(dw, want, _half_step(wt) * want.abs() + ns * U32 * (G * xh).abs().sum(0) + (G.abs() * exh).sum(0) + _tiny(wt), "dweight")
    want = G.sum(0)
    check(db, want, _half_step(wt) * want.abs() + ns * U32 * G.abs().sum(0) + _tiny(wt), "dbias")
    # each gradient alone is the same
    for i, full in enumerate((dx, dw, db)):
        part = [v.detach().requires_grad_(i == k) for k, v in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(ops.layer_norm(*part, 1e-5), part[i], dy)[0], full), i


# --------------------------------------------------------------------------------------------- squares that leave fp32's range
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
def test_grad_clip_of_values_whose_squares_leave_fp32(t):
    """Vectors of 16-bit values are added in fp32 where that is exact enough; very large and very small ones, and vectors that mix both
    with ordinary values and zeros, take the 64-bit way."""
    g = _rng(9)
    big, small = (3e4, 6e-8) if t is torch.float16 else (1e30, 1e-30)
    for values in ((big,), (small,), (big, small), (big, 1.0, 0.0), (small, 0.0), (small, 1.0), (0.0, 0.0, 0.0, small)):
        pick = torch.randint(0, len(values), (40003,), generator=g, device=_dev())
        v = (torch.tensor(values, device=_dev(), dtype=torch.float64)[pick] * (1 - 2 * (pick % 2))).to(t)
        for part in (v, v[3:], v[:7]):
            ts = part.clone()
            before = ts.double()
            want = float(before.square().sum().sqrt())
            norm = ops.GradClip([ts]).clip_(0.5 * want)
            # eight additions in fp32 of relative error 2^-24 each at most (halved by the root), then 64 bits, and one rounding
            assert abs(float(norm) - want) <= 5 * U32 * want + 2.0 ** -149, (values, float(norm), want)
            w = before * (0.5 * want / (want + 1e-6))
            check(ts, w, (_half_step(t) + 10 * U32) * w.abs() + _tiny(t), "clipped")
