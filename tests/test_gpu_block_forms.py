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
