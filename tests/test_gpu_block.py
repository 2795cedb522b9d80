"""GPU (-m gpu): the trainable block's operators -- layer_norm, linear_act, GradClip / clip_grad_norm_ -- against plain 64-bit
implementations, and a run of the three together.

Tolerances are bounds, written down before the first run: an output of type t is off by at most half a step of its type (finfo.eps / 2 of
its value) plus what 32-bit arithmetic loses on the way, counted in roundings of 2^-24 of the magnitudes that are added."""
import math

import pytest
import torch

import hopmi
from hopmi import _lib

pytestmark = pytest.mark.gpu
ops = hopmi.ops
U32 = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _dev():
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    return torch.device("cuda:0")


def _rng(seed):
    return torch.Generator(device=_dev()).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=_dev())


def _half_step(t):
    return torch.finfo(t).eps / 2


def _tiny(t):
    return torch.finfo(t).tiny * torch.finfo(t).eps          # one step of the type's subnormals


def check(got, want, tol, what=""):
    """|got - want| <= tol elementwise; equal where the 64-bit value overflows the type or is not finite."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    d = (got.double() - want).abs()
    worst = d - tol
    bad = ~(worst <= 0)
    if bad.any():
        k = int(torch.nan_to_num(worst, nan=float("inf")).flatten().argmax())
        tf = torch.broadcast_to(torch.as_tensor(tol, dtype=torch.float64, device=d.device), d.shape).flatten()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of tolerance; element {k}: got {got.flatten()[k].item():.8g} want "
                             f"{want.flatten()[k].item():.8g}, |d| {d.flatten()[k].item():.3g} > {tf[k].item():.3g}")


# ------------------------------------------------------------------------------------------------------------ layer norm
def _ln_plain(x, w, b, eps):
    mu = x.mean(-1, keepdim=True)
    r = 1 / ((x - mu).square().mean(-1, keepdim=True) + eps).sqrt()
    xh = (x - mu) * r
    return mu, r, xh, xh * w + b


# (rows, width): one element, one wave's vectors and their ends, odd widths, each form's widest row and the next (a wave: 256 vectors of
# 4 / 8 elements, 256 threads: 1024, 1024 threads: 2048, re-read rows beyond)
LN_SIZES = [(1, 1), (3, 5), (1, 64), (34, 768), (130, 1001), (2171, 33), (9, 1027), (9, 1028), (7, 2055), (7, 2056), (5, 4100), (3, 8192),
            (3, 8203), (2, 16400), (2, 40003)]


@pytest.mark.parametrize("dtype,wdtype", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32")])
@pytest.mark.parametrize("M,D", LN_SIZES)
def test_layer_norm_forward_backward(M, D, dtype, wdtype):
    t, wt = TYPES[dtype], TYPES[wdtype]
    g = _rng(M * 7919 + D)
    pad = 0 if (M + D) % 2 else 11
    buf = torch.zeros(M, D + pad, device=_dev(), dtype=t)
    buf[:, :D] = _randn(g, M, D) * (1 + 9 * (torch.rand(D, generator=g, device=_dev()) < 0.02)) + 0.7
    x = buf[:, :D].requires_grad_()
    w, b = (1 + 0.2 * _randn(g, D)).to(wt).requires_grad_(), (0.2 * _randn(g, D)).to(wt).requires_grad_()
    dy = _randn(g, M, D).to(t)
    y = ops.layer_norm(x, w, b, 1e-5)
    assert y.dtype == t and y.shape == (M, D) and y.is_contiguous()
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b, 1e-5), y)                     # the form without a tape computes the same
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    assert dx.dtype == t and dw.dtype == wt and db.dtype == wt
    again = torch.autograd.grad(ops.layer_norm(x, w, b, 1e-5), [x, w, b], dy)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, dw, db)))           # the same bits every time

    X, W, B, G = x.detach().double(), w.detach().double(), b.detach().double(), dy.double()
    mu, r, xh, want = _ln_plain(X, W, B, 1e-5)
    # roundings on the way of any one value: a thread's own additions (8 vectors of 8 at most in the register forms, D / 1024 in the
    # re-reading one), ten levels across threads, and a dozen around them
    n = 76 + D / 1024
    ax = X.abs().mean(-1, keepdim=True)
    exh = n * U32 * ((ax + X.abs()) * r + 2 * xh.abs())                          # of xh: from mu (n roundings of mean |x|), x - mu, and r
    check(y, want, _half_step(t) * want.abs() + exh * W.abs() + 2 * U32 * (xh * W).abs() + 2 * U32 * B.abs() + _tiny(t), "y")
    gw = G * W
    m0, m1 = gw.mean(-1, keepdim=True), (gw * xh).mean(-1, keepdim=True)
    want = r * (gw - m0 - xh * m1)
    em0 = n * U32 * gw.abs().mean(-1, keepdim=True)
    em1 = n * U32 * (gw * xh).abs().mean(-1, keepdim=True) + (gw.abs() * exh).mean(-1, keepdim=True)
    tol = r * (4 * U32 * gw.abs() + em0 + xh.abs() * em1 + exh * m1.abs() + 4 * U32 * (m0.abs() + (xh * m1).abs())) + n * U32 * want.abs()
    check(dx, want, _half_step(t) * want.abs() + tol + _tiny(t), "dx")
    # column sums: the rows of a wave one after the other (an even share of M over at most 512 workgroups of 4), then 4, G / 16 and 16 more
    ns = M / 1024 + 4 + 512 / 16 + 16 + 8
    want = (G * xh).sum(0)
    check(dw, want, _half_step(wt) * want.abs() + ns * U32 * (G * xh).abs().sum(0) + (G.abs() * exh).sum(0) + _tiny(wt), "dweight")
    want = G.sum(0)
    check(db, want, _half_step(wt) * want.abs() + ns * U32 * G.abs().sum(0) + _tiny(wt), "dbias")


def test_layer_norm_without_weights_partial_gradients_and_shapes():
    g = _rng(5)
    x = _randn(g, 2, 3, 50).requires_grad_()
    dy = _randn(g, 2, 3, 50)
    w, b = _randn(g, 50).requires_grad_(), _randn(g, 50).requires_grad_()
    for ww, bb in ((None, None), (w, None), (None, b), (w, b)):
        leaves = [t for t in (x, ww, bb) if t is not None]
        got = torch.autograd.grad(ops.layer_norm(x, ww, bb), leaves, dy)
        d = [t.detach().double().requires_grad_() for t in leaves]
        it = iter(d)
        args = [next(it) if t is not None else None for t in (x, ww, bb)]
        want = torch.autograd.grad(torch.nn.functional.layer_norm(args[0], (50,), args[1], args[2]), d, dy.double())
        for p, q in zip(got, want):
            check(p, q, 1e-5 * (1 + q.abs()), "gradient")                        # 1e-5 = 168 roundings of values of order one
    only_w = torch.autograd.grad(ops.layer_norm(x.detach(), w, b), [w], dy)[0]
    only_x = torch.autograd.grad(ops.layer_norm(x, w.detach(), b.detach()), [x], dy)[0]
    full = torch.autograd.grad(ops.layer_norm(x, w, b), [x, w], dy)
    assert torch.equal(only_x, full[0]) and torch.equal(only_w, full[1])
    # a gradient that is broadcast (all ones behind a sum), rows that have no common stride, a last axis that is not contiguous
    xs = _randn(g, 4, 6, 50)[:, ::2].requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.layer_norm(xs, w, b).sum(), xs)[0], torch.autograd.grad(ops.layer_norm(xs.contiguous(), w, b).sum(), xs)[0])
    xt = _randn(g, 50, 7)
    assert torch.equal(ops.layer_norm(xt.t(), w, b), ops.layer_norm(xt.t().contiguous(), w, b))
    empty = torch.zeros(0, 50, device=_dev()).requires_grad_()
    y = ops.layer_norm(empty, w, b)
    ge = torch.autograd.grad(y.sum(), [empty, w, b])
    assert y.shape == (0, 50) and ge[0].shape == (0, 50) and not ge[1].any() and not ge[2].any()
    m = ops.LayerNorm(50, device=_dev())
    m.load_state_dict(torch.nn.LayerNorm(50).state_dict())
    check(m(x), torch.nn.functional.layer_norm(x.double(), (50,)), 1e-5 * 6, "module")


def test_layer_norm_special_rows():
    """A constant row gives the bias, a NaN or an infinity stays in its own row, large offsets keep their digits."""
    g = _rng(6)
    x = _randn(g, 6, 300)
    x[1] = 3.25
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    x[4] = x[4] * 1e-3 + 1000.0
    w, b = 1 + 0.1 * _randn(g, 300), _randn(g, 300)
    y = ops.layer_norm(x, w, b)
    assert torch.equal(y[1], b) and y[2].isnan().all() and not y[3].isfinite().all()
    want = _ln_plain(x.double(), w.double(), b.double(), 1e-5)[3]
    check(y[0], want[0], 1e-5 * 6, "plain row")
    # |x| / deviation = 1e6 / (1 + the share of eps): the mean is off by up to n roundings of 1000, n = 76, against a deviation of 3.3e-3
    check(y[4], want[4], 76 * U32 * 2000 / math.sqrt(1e-6 + 1e-5) * 2, "offset row")
    check(y[5], want[5], 1e-5 * 6, "row behind")


def test_layer_norm_gradient_against_differences():
    g = _rng(7)
    x, w, b, dy = _randn(g, 5, 37), 1 + 0.1 * _randn(g, 37), _randn(g, 37), _randn(g, 5, 37)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(ops.layer_norm(*leaves), leaves, dy)
    f = lambda *a: (_ln_plain(*a, 1e-5)[3] * dy.double()).sum()
    for i, gr in enumerate(grads):
        base = [t.double() for t in (x, w, b)]
        v = _randn(g, *base[i].shape).double()
        h = 1e-5
        hi, lo = list(base), list(base)
        hi[i], lo[i] = base[i] + h * v, base[i] - h * v
        diff = (f(*hi) - f(*lo)) / (2 * h)
        # a central difference in 64 bits: h^2 third derivatives + 2^-53 / h, both below 1e-8 of the sum's terms
        assert abs(float((gr.double() * v).sum() - diff)) <= 2e-5 * float((gr.double() * v).abs().sum()) + 1e-7


# ------------------------------------------------------------------------------------------------------------ linear_act
def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z * math.sqrt(0.5))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return 0.5 * torch.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


SLOPE = {"none": 1.0, "relu": 1.0, "gelu": 1.13, "silu": 1.1}          # largest |act'|
CURVE = {"none": 0.0, "relu": 0.0, "gelu": 0.8, "silu": 0.5}           # largest |act''|
APPROX = 1e-5     # the kernels' tail polynomial (5e-6 of its value) and exp / reciprocal instructions, relative to |z| resp. to act'


def _check_linear(M, K, N, t, act, bias, res, backward, seed=0, mk=None):
    g = _rng(seed + M + 31 * K + 977 * N)
    mk = mk or (lambda *s: _randn(g, *s).to(t))
    x, w = mk(M, K).requires_grad_(backward), (mk(N, K) * K ** -0.5).to(t).detach().requires_grad_(backward)
    b = (0.5 * _randn(g, N)).to(t).requires_grad_(backward) if bias else None
    r = mk(M, N).detach().requires_grad_(backward) if res else None
    y = ops.linear_act(x, w, b, r, act)
    assert y.dtype == t and y.shape == (M, N) and y.is_contiguous()
    X, W = x.detach().double(), w.detach().double()
    B = b.detach().double() if bias else torch.zeros(N, device=_dev(), dtype=torch.float64)
    R = r.detach().double() if res else torch.zeros((), device=_dev(), dtype=torch.float64)
    z = X @ W.t() + B
    # z: K + 1 additions, each rounded (or, inside the matrix unit, cut) to at most one step of 2^-23 of the magnitudes added
    ez = (K + 2) * 2 * U32 * (X.abs() @ W.abs().t() + B.abs())
    want = _act(z, act) + R
    u = _half_step(t)
    check(y, want, u * want.abs() + SLOPE[act] * ez + APPROX * z.abs() + 2 * U32 * R.abs() + _tiny(t), f"y {M}x{K}x{N} {act}")
    if not backward:
        return
    dy = _randn(g, M, N).to(t)
    leaves = [v for v in (x, w, b, r) if v is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    assert all(p.dtype == t and p.shape == v.shape for p, v in zip(grads, leaves))
    G = dy.double()
    dz = G * _act_grad(z, act)
    # act' is taken at z rounded to t; the unrounded dz feeds the bias gradient, the rounded one the products
    e0 = G.abs() * (CURVE[act] * (u * z.abs() + ez) + 2 * APPROX * (1 + z.abs()) + _tiny(t)) + 2 * U32 * dz.abs()
    if act == "relu":
        e0 = e0 + torch.where(z.abs() <= ez + _tiny(t), G.abs(), torch.zeros_like(G))      # the kink: either side is right
    e1 = e0 + u * (dz.abs() + e0) + _tiny(t)
    want = dz @ W
    check(grads[0], want, u * want.abs() + e1 @ W.abs() + (N + 2) * 2 * U32 * ((dz.abs() + e1) @ W.abs()) + _tiny(t), "dx")
    want = dz.t() @ X
    check(grads[1], want, u * want.abs() + e1.t() @ X.abs() + (M + 2) * 2 * U32 * ((dz.abs() + e1).t() @ X.abs()) + _tiny(t), "dw")
    if bias:
        want = dz.sum(0)
        check(grads[2], want, u * want.abs() + e0.sum(0) + (M + 2) * U32 * (dz.abs() + e0).sum(0) + _tiny(t), "db")
    if res:
        assert torch.equal(grads[-1], dy)
    if act != "relu":
        again = torch.autograd.grad(ops.linear_act(x, w, b, r, act), leaves, dy)
        assert all(torch.equal(p, q) for p, q in zip(grads, again))              # the same bits every time


# few rows (each number of 16-row blocks, odd contraction ends), the first row counts of the tiled form, odd sides, one and several
# k-steps, contraction tails (64 n + 8 m and odd), split contractions, one column
LIN_SIZES = [(64, 4096, 72), (48, 4096, 4096), (33, 2048, 136), (1, 1, 1), (1, 768, 2304), (2, 3, 5), (16, 33, 17), (17, 64, 16), (33, 129, 40), (34, 768, 768), (64, 130, 50), (64, 4096, 19),
             (65, 64, 64), (65, 72, 40), (66, 7, 9), (129, 100, 33), (100, 1, 130), (300, 1021, 427), (512, 768, 256), (130, 4160, 136),
             (1000, 200, 1), (260, 4352, 200), (1024, 1024, 1030), (2176, 768, 770)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("M,K,N", LIN_SIZES)
def test_linear_act_sizes(M, K, N, dtype):
    _check_linear(M, K, N, TYPES[dtype], "gelu", True, True, True)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("bias,res", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("M,K,N", [(5, 40, 24), (200, 136, 72), (130, 50, 35)])
def test_linear_act_epilogues(M, K, N, bias, res, act, dtype):
    _check_linear(M, K, N, TYPES[dtype], act, bias, res, True)


@pytest.mark.parametrize("M,K,N", [(4000, 72, 3600), (3585, 320, 3992), (72, 4000, 264)])
def test_linear_act_large_tiles(M, K, N):
    """Results of 224 and more tiles of 256 x 256 (ragged ones), in each of the three products."""
    _check_linear(M, K, N, torch.bfloat16, "gelu", True, True, True)


def test_linear_act_large_weight_gradient():
    _check_linear(200, 3600, 4008, torch.float16, "none", True, False, True)


# backward products that share a launch: either one first, splits in either contraction, sums of one and of many row groups, ragged sides
PAIRED = [(4352, 768, 2304), (2171, 1021, 427), (300, 1021, 427), (4000, 72, 3600), (16000, 40, 40), (16000, 768, 72), (65, 72, 1200),
          (8192, 1024, 1024), (4352, 768, 768), (128, 4096, 4096), (70, 1, 2000), (3000, 2000, 1)]


@pytest.mark.parametrize("dtype,act,bias", [("bf16", "gelu", True), ("fp16", "none", True), ("bf16", "silu", False)])
@pytest.mark.parametrize("M,K,N", PAIRED)
def test_linear_act_both_products(M, K, N, dtype, act, bias):
    _check_linear(M, K, N, TYPES[dtype], act, bias, False, True)


def test_linear16_bwd_entry_point():
    """Both products and the bias gradient's sums by one C call, and nothing written next to them."""
    L, t = _lib.lib(), torch.bfloat16
    g = _rng(77)
    st = torch.cuda.current_stream().cuda_stream
    for M, K, N in ((65, 72, 40), (300, 1024, 432), (34, 768, 768), (2176, 768, 776)):
        dz, w, x = _randn(g, M, N).to(t), _randn(g, N, K).to(t), _randn(g, M, K).to(t)
        out = torch.full((M * K + N * K + N + 24,), 7.0, device=_dev(), dtype=t)
        dx, dw, db = out[8:8 + M * K], out[16 + M * K:16 + M * K + N * K], out[24 + M * K + N * K:]
        part = torch.empty(L.hopmi_act_bwd16_ws_floats(M, N), device=_dev())
        ws = torch.empty(max(1, L.hopmi_linear16_bwd_ws_floats(M, N, K)), device=_dev())
        assert L.hopmi_act_bwd16(dz.data_ptr(), N, None, 0, None, 0, None, part.data_ptr(), 0, M, N, 1, st) == 0
        assert L.hopmi_linear16_bwd(dz.data_ptr(), N, w.data_ptr(), K, x.data_ptr(), K, dx.data_ptr(), dw.data_ptr(), part.data_ptr(),
                                    db.data_ptr(), M, N, K, 1, ws.data_ptr(), st) == 0
        D, W, X = dz.double(), w.double(), x.double()
        for got, a, b, n in ((dx.view(M, K), D, W, N), (dw.view(N, K), D.t(), X, M)):
            want = a @ b
            check(got, want, _half_step(t) * want.abs() + (n + 2) * 2 * U32 * (a.abs() @ b.abs()) + _tiny(t), f"{M}x{K}x{N}")
        check(db, D.sum(0), _half_step(t) * D.sum(0).abs() + (M + 2) * U32 * D.abs().sum(0) + _tiny(t), "db")
        gaps = torch.cat([out[:8], out[8 + M * K:16 + M * K], out[16 + M * K + N * K:24 + M * K + N * K]])
        assert (gaps == 7.0).all()


def test_linear_act_operands_as_they_lie():
    """Row strides, offsets that break the alignment, a transposed operand, leading axes, broadcast residuals and gradients."""
    g = _rng(11)
    t = torch.bfloat16
    for M, K, N in ((40, 64, 48), (150, 64, 48), (150, 61, 45)):
        x, w, r = _randn(g, M, K).to(t), (_randn(g, N, K) / 8).to(t), _randn(g, M, N).to(t)
        want = ops.linear_act(x, w, None, r, "silu")
        big = torch.zeros(M, K + 13, device=_dev(), dtype=t)
        for off in (0, 1, 8):
            v = big[:, off:off + K]
            v.copy_(x)
            assert torch.equal(ops.linear_act(v, w, None, r, "silu"), want)
        bw, br = torch.zeros(N, K + 5, device=_dev(), dtype=t), torch.zeros(M, N + 3, device=_dev(), dtype=t)
        bw[:, 3:3 + K], br[:, 1:1 + N] = w, r
        assert torch.equal(ops.linear_act(x, bw[:, 3:3 + K], None, br[:, 1:1 + N], "silu"), want)
        assert torch.equal(ops.linear_act(x.t().contiguous().t(), w.t().contiguous().t(), None, r, "silu"), want)
        assert torch.equal(ops.linear_act(x.view(2, M // 2, K), w, None, r.view(2, M // 2, N), "silu"), want.view(2, M // 2, N))
        # a residual row for all rows: its gradient is the sum over them
        row = r[:1].clone().requires_grad_()
        xx = x.clone().requires_grad_()
        y = ops.linear_act(xx, w, None, row, "none")
        assert torch.equal(y, ops.linear_act(x, w, None, row.detach().expand(M, N).contiguous()))
        dy = _randn(g, M, N).to(t)
        gx, gr = torch.autograd.grad(y, [xx, row], dy)
        wr = dy.double().sum(0, keepdim=True)
        # torch's reduction of the broadcast axis: fp32 sums, rounded to bf16
        check(gr, wr, _half_step(t) * wr.abs() + M * U32 * dy.double().abs().sum(0, keepdim=True), "broadcast residual")
        # a gradient that is itself broadcast
        ones = torch.autograd.grad(ops.linear_act(xx, w, None, r, "gelu").sum(), xx)[0]
        assert torch.equal(ones, torch.autograd.grad(ops.linear_act(xx, w, None, r, "gelu"), xx, torch.ones(M, N, device=_dev(), dtype=t))[0])


def test_linear_act_partial_gradients_and_empty_batches():
    g = _rng(12)
    t = torch.float16
    x, w, b = _randn(g, 100, 72).to(t), (_randn(g, 56, 72) / 8).to(t), _randn(g, 56).to(t)
    dy = _randn(g, 100, 56).to(t)
    for act in ("none", "gelu"):
        full = [v.clone().requires_grad_() for v in (x, w, b)]
        want = torch.autograd.grad(ops.linear_act(*full, activation=act), full, dy)
        for i in range(3):
            part = [v.clone().requires_grad_(i == k) for k, v in enumerate((x, w, b))]
            assert torch.equal(torch.autograd.grad(ops.linear_act(*part, activation=act), part[i], dy)[0], want[i])
    e = torch.zeros(0, 72, device=_dev(), dtype=t).requires_grad_()
    lw, lb = w.clone().requires_grad_(), b.clone().requires_grad_()
    y = ops.linear_act(e, lw, lb, activation="gelu")
    ge = torch.autograd.grad(y.sum(), [e, lw, lb])
    assert y.shape == (0, 56) and ge[0].shape == (0, 72) and not ge[1].any() and not ge[2].any()


def test_linear_act_special_values():
    """Infinities and NaN stay in their rows, large and tiny values go through the activations as their limits say."""
    t = torch.bfloat16
    for M in (8, 100):
        z = torch.tensor([0.0, -0.0, 1e-30, 5.0, -5.0, 12.0, -12.0, 90.0, -90.0, 3e4, -3e4, 1e38, -1e38, float("inf"), float("-inf"), float("nan")],
                         device=_dev()).to(t)
        n = z.numel()
        x = torch.zeros(M, 16, device=_dev(), dtype=t)
        x[:, 0] = 1
        w = torch.zeros(n, 16, device=_dev(), dtype=t)
        for act in ("relu", "gelu", "silu"):
            y = ops.linear_act(x, w, z, None, act).double()
            want = _act(z.double(), act)
            want[-2] = 0.0                                                      # the limit at -inf
            fin = want.isfinite()
            check(y[:, fin], want[fin].expand(M, -1), _half_step(t) * want[fin].abs() + APPROX * want[fin].abs() + _tiny(t), act)
            assert (y[:, n - 3] == float("inf")).all() and y[:, n - 1].isnan().all()
            zz = z.clone().requires_grad_()
            gz = torch.autograd.grad(ops.linear_act(x, w, zz, None, act), zz, torch.ones(M, n, device=_dev(), dtype=t))[0].double() / M
            wg = _act_grad(z.double(), act)
            wg[-2], wg[-3] = 0.0, 1.0
            check(gz[:-1], wg[:-1], 2 * _half_step(t) * wg[:-1].abs() + 2 * APPROX + 1e-6, act + " gradient")
        xb = x.clone()
        xb[3, 1] = float("nan")
        yb = ops.linear_act(xb, torch.ones_like(w), None, None, "gelu")
        assert yb[3].isnan().all() and yb[:3].isfinite().all() and yb[4:].isfinite().all()


def test_linear_act_refusals_on_device():
    x, w = torch.zeros(4, 8, device=_dev(), dtype=torch.bfloat16), torch.zeros(6, 8, device=_dev(), dtype=torch.bfloat16)
    for call, word in ((lambda: ops.linear_act(x.float(), w.float()), "ops.linear"), (lambda: ops.linear_act(x, w.half()), "one type"),
                       (lambda: ops.linear_act(x, w[:, :7]), "do not fit"), (lambda: ops.linear_act(x[:, :0], w[:, :0]), "empty side"),
                       (lambda: ops.linear_act(x, w, w[0]), "bias has shape"), (lambda: ops.linear_act(x, w, None, x), "broadcast"),
                       (lambda: ops.linear_act(x, w.cpu()), "is on cpu"), (lambda: ops.layer_norm(x, w[0].cpu()), "is on cpu"),
                       (lambda: ops.layer_norm(x, w[0].half()), "that type, or fp32"), (lambda: ops.layer_norm(x, w[0], w[0].float()), "one type for both"),
                       (lambda: ops.layer_norm(x, w[0, :7]), "shape"), (lambda: ops.layer_norm(x, eps=float("nan")), "eps")):
        with pytest.raises(_lib.HopmiError, match=word):
            call()
    with torch.autocast("cuda", dtype=torch.bfloat16):                           # fp32 operands take the autocast type
        xf = torch.randn(70, 8, device=_dev()).requires_grad_()
        y = ops.linear_act(xf, w.float())
        assert y.dtype == torch.bfloat16 and torch.autograd.grad(y.sum(), xf)[0].dtype == torch.float32


def test_gradients_of_gradients_are_refused_where_they_are_taken():
    """Under create_graph the first gradients are right; going through them again is an error, not a silent zero."""
    g = _rng(13)
    x, w = _randn(g, 80, 24).requires_grad_(), _randn(g, 24).requires_grad_()
    y = ops.layer_norm(x, w)
    first = torch.autograd.grad(y.sum(), [x, w], create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(first, torch.autograd.grad(ops.layer_norm(x, w).sum(), [x, w])))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(first[0].square().sum(), x)
    xb, wb = x.detach().bfloat16().requires_grad_(), _randn(g, 16, 24).bfloat16().requires_grad_()
    gb = torch.autograd.grad(ops.linear_act(xb, wb, activation="gelu").sum(), [xb, wb], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(gb[0].float().square().sum(), xb)
    # an operand changed between the passes is noticed
    y = ops.layer_norm(x, w)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)


# ------------------------------------------------------------------------------------------------------------ GradClip
def _clip_case(seed, count, dtypes, scale=1.0, odd=True):
    g = _rng(seed)
    out = []
    for i in range(count):
        n = 1 + int(torch.randint(0, 40000 if i % 9 == 0 else 700, (1,), generator=g, device=_dev()))
        base = (_randn(g, n + 3) * scale).to(TYPES[dtypes[i % len(dtypes)]])
        out.append(base[i % 3 if odd else 0:][:n])                               # some off the allocator's alignment
    return out


@pytest.mark.parametrize("dtypes", [["fp32"], ["bf16"], ["fp16"], ["fp32", "bf16", "fp16"]])
@pytest.mark.parametrize("count", [1, 7, 119, 120, 121, 164, 165, 166, 250, 251, 300])
@pytest.mark.parametrize("into", [False, True])
def test_grad_clip_norm_and_values(count, dtypes, into):
    for limit in (0.5, 1e6, 0.0):
        ts = _clip_case(count, count, dtypes)
        before = [t.clone() for t in ts]
        outs = [torch.full(t.shape, 7.0, device=_dev()) for t in ts] if into else None
        norm = ops.GradClip(ts, out=outs).clip_(limit)
        want = math.sqrt(sum(float(t.double().square().sum()) for t in before))
        assert norm.dtype == torch.float32 and norm.shape == () and abs(float(norm) - want) <= 2 * U32 * want
        c = min(1.0, limit / (want + 1e-6))
        for t, b, o in zip(ts, before, outs or ts):
            if into:
                assert torch.equal(t, b)
            w = b.double() * c
            # c is rounded to fp32, the product once more, then the type's own half step
            check(o, w, (_half_step(o.dtype) + 3 * U32) * w.abs() + _tiny(o.dtype), "clipped")
            if c == 1.0 and not into:
                assert torch.equal(t, b)


def test_grad_clip_leaves_neighbours_alone():
    flat = torch.ones(5000, device=_dev())
    parts = [flat[3:1000], flat[1001:1002], flat[1010:4321]]
    ops.GradClip(parts).clip_(1.0)
    out = torch.ones(5000, dtype=torch.bool, device=_dev())
    for a, b in ((3, 1000), (1001, 1002), (1010, 4321)):
        out[a:b] = False
    assert (flat[out] == 1).all() and (flat[~out] < 1).all()


def test_grad_clip_special_values_and_shapes():
    dev = _dev()
    big = [torch.full((1000,), 1e30, device=dev), torch.zeros(0, device=dev), torch.full((2, 3), -2e30, device=dev)]
    want = math.sqrt(1000 * 1e60 + 6 * 4e60)                                    # its square is far beyond fp32
    n = ops.GradClip(big).clip_(1.0)
    assert abs(float(n) - want) <= 2 * U32 * want and abs(float(big[0][0]) - 1e30 / want) <= 4 * U32 * 1e30 / want
    tiny = [torch.full((64,), 1e-30, device=dev)]
    assert abs(float(ops.GradClip(tiny).clip_(1.0)) - 8e-30) <= 2 * U32 * 8e-30
    for bad, c_finite in ((float("nan"), float("nan")), (float("inf"), 0.0)):
        t = torch.ones(300, device=dev)
        t[17] = bad
        m = ops.GradClip([t]).clip_(1.0)
        if bad != bad:
            assert m.isnan() and t.isnan().all()
        else:
            assert m == float("inf") and t[17].isnan() and (t[:17] == 0).all()
    t = torch.full((300,), 2.0, device=dev)
    assert abs(float(ops.GradClip([t]).clip_(float("inf"))) - 2 * math.sqrt(300)) < 1e-4 and (t == 2).all()
    zero = torch.zeros(10, device=dev)
    assert float(ops.GradClip([zero, torch.zeros(0, 4, device=dev)]).clip_(1.0)) == 0.0
    assert float(ops.GradClip([torch.zeros(0, device=dev)]).clip_(1.0)) == 0.0
    perm = torch.ones(4, 5, 6, device=dev).permute(2, 0, 1)                     # dense in another order of its axes
    o = torch.empty_like(perm)
    assert o.stride() == perm.stride()
    ops.GradClip([perm], out=[o]).clip_(1.0)
    check(o, torch.full((6, 4, 5), 1 / math.sqrt(120), device=dev, dtype=torch.float64), 4 * U32, "permuted")
    for bad, word in (([t[::2]], "without gaps"), ([t, t], "share memory"), ([t, t[5:9]], "share memory"), ([t.double()], "fp32, bf16 or fp16"),
                      ([t, torch.zeros(3)], "is on cpu")):
        with pytest.raises(_lib.HopmiError, match=word):
            ops.GradClip(bad)
    for o, word in (([t], "share memory"), ([t.new_zeros(299)], "shape and strides"), ([t.new_zeros(300).half()], "fp32 tensor"), ([], "outputs for")):
        with pytest.raises(_lib.HopmiError, match=word):
            ops.GradClip([t], out=o)
    with pytest.raises(_lib.HopmiError, match="max_norm"):
        ops.GradClip([t]).clip_(-1.0)


def test_clip_grad_norm_is_torchs():
    g = _rng(21)
    ps = [torch.nn.Parameter(_randn(g, *s)) for s in ((64, 33), (7,), (5, 3, 2), (1,))] + [torch.nn.Parameter(_randn(g, 4))]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, q in zip(ps[:-1], qs):
        p.grad = _randn(g, *p.shape)
        q.grad = p.grad.clone()
    v = ps[0].grad._version
    a, b = ops.clip_grad_norm_(ps, 0.7), torch.nn.utils.clip_grad_norm_(qs, 0.7)
    # torch: 32-bit sums of at most 2112 squares in pairs and a 32-bit factor
    assert abs(float(a) - float(b)) <= 64 * U32 * float(b) and ps[-1].grad is None and ps[0].grad._version > v
    for p, q in zip(ps[:-1], qs):
        check(p.grad, q.grad.double(), 70 * U32 * q.grad.double().abs(), "gradient")


# ------------------------------------------------------------------------------------------- streams, graphs, a run of the three
def _block(dev, t, D=72, H=136, rows=150, seed=31):
    g = _rng(seed)
    p = dict(g=(1 + 0.1 * _randn(g, D)), b=0.1 * _randn(g, D), w1=_randn(g, H, D) * D ** -0.5, b1=0.1 * _randn(g, H), w2=_randn(g, D, H) * H ** -0.5,
             b2=0.1 * _randn(g, D))
    return {k: v.to(t) for k, v in p.items()}, _randn(g, rows, D).to(t), _randn(g, rows, D).to(t)


def _block_forward(p, x):
    """A pre-norm residual block: x + W2 gelu(W1 norm(x) + b1) + b2."""
    h = ops.layer_norm(x, p["g"], p["b"])
    return ops.linear_act(ops.linear_act(h, p["w1"], p["b1"], activation="gelu"), p["w2"], p["b2"], residual=x)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_block_step_against_64_bits(dtype):
    """Forward, backward, clipping into fp32 and the one-launch Adam step of a block, against the same in 64 bits."""
    t = TYPES[dtype]
    p, x, dy = _block(_dev(), t)
    leaves = {k: v.clone().requires_grad_() for k, v in p.items()}
    xl = x.clone().requires_grad_()
    y = _block_forward(leaves, xl)
    grads = torch.autograd.grad(y, [xl, *leaves.values()], dy)
    y = y.detach()
    d = {k: v.double().requires_grad_() for k, v in p.items()}
    xd = x.double().requires_grad_()
    f = torch.nn.functional
    yd = xd + f.linear(f.gelu(f.linear(f.layer_norm(xd, (xd.shape[1],), d["g"], d["b"]), d["w1"], d["b1"])), d["w2"], d["b2"])
    want = torch.autograd.grad(yd, [xd, *d.values()], dy.double())
    # independent roundings, four on the longest way (norm, hidden, its gradient, dz) and the result's own: norms of the differences
    # against norms of the values, each rounding at most half a step
    lim = 6 * _half_step(t)
    for n, a, b in zip(["y", "x", *p], [y, *grads], [yd.detach(), *want]):
        assert float((a.double() - b).norm() / b.norm()) <= lim, n
    masters = [v.float() for v in p.values()]
    main = [torch.empty_like(m) for m in masters]
    norm = ops.GradClip(list(grads[1:]), out=main).clip_(1.0)
    wn = math.sqrt(sum(float(v.double().square().sum()) for v in grads[1:]))
    assert abs(float(norm) - wn) <= 2 * U32 * wn
    m1, m2 = [torch.zeros_like(m) for m in masters], [torch.zeros_like(m) for m in masters]
    plan = ops.AdamPlan(masters, m1, m2)
    plan.bind(main, m1, m2)
    start = [m.clone() for m in masters]
    plan.step(1e-2, 0.9, 0.999, 1e-8, torch.ones((), device=_dev()))
    for m, s, gr in zip(masters, start, grads[1:]):
        c = min(1.0, 1.0 / (wn + 1e-6))
        step = 1e-2 * (gr.double() * c) / ((gr.double() * c).abs() + 1e-8)       # the first Adam step, bias corrections cancelling
        check(m, s.double() - step, 1e-2 * 1e-4 + 2 * U32 * s.double().abs(), "Adam step")


def test_block_on_another_stream_and_two_at_once():
    p, x, dy = _block(_dev(), torch.bfloat16)
    want = _block_forward(p, x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for k in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(_block_forward(p, x))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want) for v in got)


def test_block_step_captured_and_replayed():
    """A whole step (forward, backward, clip) recorded into a graph, replayed with eager work in between; and two recordings that replay
    at once on two streams, each with workspaces of its own."""
    def record(seed):
        p, x, dy = _block(_dev(), torch.bfloat16, D=768, H=520, rows=300, seed=seed)
        leaves = {k: v.clone().requires_grad_() for k, v in p.items()}
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        out = {}
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            with torch.cuda.graph(gr, stream=s):
                y = _block_forward(leaves, x)
                g = torch.autograd.grad(y, list(leaves.values()), dy)
                main = [torch.empty(v.shape, device=v.device) for v in g]
                norm = ops.GradClip(list(g), out=main).clip_(0.25)
                out["r"] = [y, norm, *g, *main]
        torch.cuda.current_stream().wait_stream(s)
        return gr, leaves, x, dy, out["r"]

    def eager(leaves, x, dy):
        ll = {k: v.detach().clone().requires_grad_() for k, v in leaves.items()}
        y = _block_forward(ll, x)
        g = torch.autograd.grad(y, list(ll.values()), dy)
        main = [torch.empty(v.shape, device=v.device) for v in g]
        norm = ops.GradClip(list(g), out=main).clip_(0.25)
        return [v.detach() for v in [y, norm, *g, *main]]

    ops.linear_act(torch.zeros(300, 768, device=_dev(), dtype=torch.bfloat16), torch.zeros(520, 768, device=_dev(), dtype=torch.bfloat16))
    a, b = record(41), record(42)
    for k in range(4):
        for gr, leaves, x, dy, r in (a, b):
            x.copy_(torch.randn(x.shape, device=x.device, generator=_rng(100 + k)))
        want = [eager(leaves, x, dy) for _, leaves, x, dy, _ in (a, b)]
        torch.cuda.synchronize()
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        for s, (gr, *_) in zip((s1, s2), (a, b)):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for w, (*_, r) in zip(want, (a, b)):
            assert all(torch.equal(p, q) for p, q in zip(w, r)), k


@pytest.mark.parametrize("recorded", [False, True])
def test_training_step_clips_by_max_grad_norm(recorded, monkeypatch):
    """args.max_grad_norm: train_llm, eager and recorded, steps on gradients of that global norm (the gradients that a step leaves behind
    are the ones its optimizer read), and a limit above the norm changes no bit."""
    import copy
    from oracle.golden_util import Accel, step_args
    from test_gpu_graph import _deterministic_draws, _pair
    _deterministic_draws(monkeypatch)
    m0, d0, inp = _pair(9, _dev())
    batch = (inp["in_audio"], inp["log_melspec"], inp["text"], inp["target_dir_vec"], inp["vid_indices"])

    def steps(limit, n):
        m, d = copy.deepcopy(m0), copy.deepcopy(d0)
        m._randn_like = m0._randn_like
        g = torch.optim.Adam([p for p in m.parameters() if p.requires_grad], lr=1e-4, betas=(0.5, 0.999))
        o = torch.optim.Adam(d.parameters(), lr=1e-4, betas=(0.5, 0.999))
        args = step_args(9)
        if limit is not None:
            args.max_grad_norm = limit
        run = hopmi.GraphedTrainStep(args, m, d, g, o, eager_calls=1) if recorded else lambda e, *b: hopmi.train_llm(args, e, *b, m, d, g, o, Accel())
        for _ in range(n):
            run(0, *batch)
        torch.cuda.synchronize()
        grads = [p.grad for p in m.parameters() if p.grad is not None]
        assert grads and (not recorded or run.n_replay == n - 1)
        return m, math.sqrt(sum(float(v.double().square().sum()) for v in grads))

    free, norm = steps(None, 3)
    same, _ = steps(1e6 * norm, 3)
    assert all(torch.equal(p, q) for p, q in zip(free.parameters(), same.parameters()))
    clipped, after = steps(0.125 * norm, 3)
    # every step's norm stays far above the limit here, so the last step's gradients have it as their norm: 1e-6 in the formula's
    # denominator and one rounding per value
    assert abs(after - 0.125 * norm) <= 1e-5 * norm
    assert not all(torch.equal(p, q) for p, q in zip(free.parameters(), clipped.parameters()))



# --------------------------------------------------------------------------------------------------------- far offsets, wide strides
def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: the last rows are as right as the first."""
    t = torch.bfloat16
    g = _rng(61)
    D, M = 1024, (1 << 21) + 5
    x = torch.zeros(M, D, device=_dev(), dtype=t)
    w, b = (1 + 0.1 * _randn(g, D)).to(t), (0.1 * _randn(g, D)).to(t)
    ends = torch.tensor([0, 1, M - 2, M - 1], device=_dev())
    x[ends] = _randn(g, 4, D).to(t)
    y = ops.layer_norm(x, w, b)
    want = _ln_plain(x[ends].double(), w.double(), b.double(), 1e-5)[3]
    check(y[ends], want, _half_step(t) * want.abs() + 1e-5 * (1 + want.abs()), "layer norm")        # 1e-5: 160 roundings of values of order one
    assert torch.equal(y[2:-2], b.expand(M - 4, D))
    del y
    # the same rows through a product with as many results, and its input gradient
    wl = (_randn(g, 1032, D) / 32).to(t)
    xl = x.requires_grad_()
    y = ops.linear_act(xl, wl)
    want = x[ends].detach().double() @ wl.double().t()
    check(y[ends], want, _half_step(t) * want.abs() + (D + 2) * 2 * U32 * (x[ends].detach().double().abs() @ wl.double().abs().t()) + _tiny(t), "linear")
    dy = torch.zeros_like(y)
    dy[ends] = _randn(g, 4, 1032).to(t)
    del y
    dx = torch.autograd.grad(ops.linear_act(xl, wl), xl, dy)[0]
    want = dy[ends].double() @ wl.double()
    check(dx[ends], want, _half_step(t) * want.abs() + 1034 * 2 * U32 * (dy[ends].double().abs() @ wl.double().abs()) + _tiny(t), "linear dx")
    assert not dx[2:-2].any()
    del dy, dx
    flat = x.detach().view(-1)
    flat.fill_(0.5)
    n = ops.GradClip([flat[3:]]).clip_(1.0)
    want = 0.5 * math.sqrt(M * D - 3)
    assert abs(float(n) - want) <= 2 * U32 * want
    v = 0.5 / (want + 1e-6)
    assert (flat[:3] == 0.5).all() and (flat[3:].float() - v).abs().max() <= (_half_step(t) + 4 * U32) * v


def test_wide_strides():
    """Rows further apart than a tile's 32-bit offsets reach: read where they are by the few-row form, copied for the tiles."""
    t = torch.float16
    g = _rng(62)
    ld = (1 << 22) + 24
    buf = torch.zeros(70, ld, device=_dev(), dtype=t)
    w = (_randn(g, 40, 96) / 10).to(t)
    for M in (3, 70):
        x = _randn(g, M, 96).to(t)
        v = buf[:M, 8:104]
        v.copy_(x)
        assert torch.equal(ops.linear_act(v, w, activation="relu"), ops.linear_act(x, w, activation="relu"))
        assert torch.equal(ops.layer_norm(v), ops.layer_norm(x))
        a, c = v.detach().requires_grad_(), x.clone().requires_grad_()
        dy = _randn(g, M, 40).to(t)
        assert torch.equal(torch.autograd.grad(ops.linear_act(a, w), a, dy)[0], torch.autograd.grad(ops.linear_act(c, w), c, dy)[0])


def test_grad_clip_plan_follows_its_tensors():
    dev = _dev()
    t, u = torch.full((1000,), 3.0, device=dev), torch.full((10, 10), 4.0, device=dev)
    plan = ops.GradClip([t, u])
    want = math.sqrt(9000 + 1600)
    assert abs(float(plan.clip_(1e9)) - want) <= 2 * U32 * want
    t.data = torch.full((1000,), 1.0, device=dev)                                # another piece of memory behind the same tensor
    want = math.sqrt(1000 + 1600)
    assert abs(float(plan.clip_(1.0)) - want) <= 2 * U32 * want and (t < 0.1).all() and (u < 0.1).all()
    u.data = torch.zeros(3, device=dev)
    with pytest.raises(_lib.HopmiError, match="any more"):
        plan.clip_(1.0)
    # two calls in flight on two streams, each with sums of its own
    big = [torch.full((5_000_000,), float(k + 1), device=dev) for k in range(2)]
    torch.cuda.synchronize()
    norms = []
    for k in range(2):
        with torch.cuda.stream(torch.cuda.Stream()):
            norms.append(ops.GradClip([big[k]]).clip_(float("inf")))
    torch.cuda.synchronize()
    for k in range(2):
        want = (k + 1) * math.sqrt(5_000_000)
        assert abs(float(norms[k]) - want) <= 2 * U32 * want


def test_grad_clip_plan_looks_at_moved_tensors_again():
    """Memory behind a plan's tensors may be exchanged: what the plan refused at first it refuses then too, before any launch."""
    dev = _dev()
    t, u, o = torch.ones(1000, device=dev), torch.ones(1000, device=dev), torch.zeros(1000, device=dev)
    plan, into = ops.GradClip([t, u]), ops.GradClip([u], out=[o])
    both = torch.full((1500,), 2.0, device=dev)
    keep = u.data
    t.data, u.data = both[:1000], both[500:]
    for _ in range(2):                                       # (not only the first time)
        with pytest.raises(_lib.HopmiError, match="share memory"):
            plan.clip_(1.0)
    u.data = torch.ones(2000, device=dev)[::2]
    with pytest.raises(_lib.HopmiError, match="without gaps"):
        plan.clip_(1.0)
    u.data = torch.ones(1000)
    for p in (plan, into):
        with pytest.raises(_lib.HopmiError, match="is on cpu"):
            p.clip_(1.0)
    u.data, o.data = keep, torch.zeros(999, device=dev)
    with pytest.raises(_lib.HopmiError, match="shape"):
        into.clip_(1.0)
    want = math.sqrt(1000 * 4 + 1000)
    assert abs(float(plan.clip_(1e9)) - want) <= 2 * U32 * want
    assert (both == 2).all() and (u == 1).all()
