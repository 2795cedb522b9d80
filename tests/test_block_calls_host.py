"""CPU: the trainable block's operators inside the training steps, and what their modules refuse."""
import types

import pytest
import torch

import hopmi
from hopmi import _lib

ops = hopmi.ops


def test_recorded_step_over_ranks_refuses_a_limit_that_is_set_later(tmp_path):
    """`args` may change after construction: the refusal comes with the call, before anything is enqueued."""
    import torch.distributed as dist
    mod = torch.nn.Linear(2, 2)
    if dist.is_initialized():
        pytest.skip("a process group is up in this process")
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        args = types.SimpleNamespace(loss_gan_weight=0.0)
        run = hopmi.GraphedTrainStep(args, mod, mod, None, None, force_exchange=True)
        args.max_grad_norm = 1.0
        on_device = types.SimpleNamespace(is_cuda=True)                          # (all that is looked at before the refusal)
        with pytest.raises(_lib.HopmiError, match="max_grad_norm"):
            run(0, on_device, None, None, None, None)
        assert run.n_eager == 0 and run.eager_left == {}
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("affine", [False, True])
def test_layer_norm_module_refuses_another_width(affine):
    """Without weights the operator itself cannot tell: it normalises over whatever the last axis is."""
    m = ops.LayerNorm(8, elementwise_affine=affine)
    for shape in ((4, 16), (8, 1), ()):
        with pytest.raises(_lib.HopmiError, match="normalized_shape"):
            m(torch.zeros(shape))
    with pytest.raises(_lib.HopmiError, match="no CPU fallback"):
        m(torch.zeros(4, 8))


# ------------------------------------------------------------------------------------------- clipping inside the training steps
class _Generator(torch.nn.Module):
    """The generators' call shapes (train_llm's and train_iter_gan's: the poses come out of the last audio-shaped operand)."""

    def __init__(self, poses):
        super().__init__()
        self.lin, self.poses = torch.nn.Linear(4, poses), poses

    def forward(self, *operands):
        out = self.lin(operands[0] if operands[0].shape[-1] == 4 else operands[2])
        return out, out.mean(1), None, None


class _Scores(torch.nn.Module):
    def __init__(self, poses):
        super().__init__()
        self.lin = torch.nn.Linear(poses, 1)

    def forward(self, poses, text=None):
        return torch.sigmoid(self.lin(poses).mean(1))

    def update_statistics(self, poses):
        pass


class _Optim:
    """An SGD optimizer that takes the loss's scale out of the gradients, unless that has been done, and writes down what it steps on."""

    def __init__(self, module, name, log, scale=1.0):
        self.opt, self.name, self.log, self.scale, self.scaled = torch.optim.SGD(module.parameters(), lr=0.1), name, log, scale, True
        self.param_groups = self.opt.param_groups

    def zero_grad(self):
        self.opt.zero_grad()

    def unscale(self):
        for g in self.param_groups:
            for p in g["params"]:
                p.grad.div_(self.scale)
        self.scaled = False

    def step(self):
        if self.scaled:
            self.unscale()
        self.scaled = True
        self.log.append(("step", self.name, [p.grad.clone() for g in self.param_groups for p in g["params"]]))
        self.opt.step()


def _trace(monkeypatch, log):
    """The device operator's place is taken by torch's: what is looked at here is what it is given, and when."""
    from hopmi import steps

    def clip(params, limit):
        params = list(params)
        log.append(("clip", params, limit))
        return torch.nn.utils.clip_grad_norm_(params, limit)

    monkeypatch.setattr(steps._ops, "clip_grad_norm_", clip)
    monkeypatch.setattr(steps, "FUSED_LOSSES", False)


def _args(**more):
    return types.SimpleNamespace(loss_regression_weight=600.0, loss_gan_weight=5.0, loss_kld_weight=0.0, loss_reg_weight=0.0, z_type="none",
                                 loss_warmup=0, n_pre_poses=4, **more)


def _norm(ts):
    return float(torch.cat([t.reshape(-1) for t in ts]).norm())


def _llm(args, epoch, accelerator, log):
    torch.manual_seed(3)
    g, d = _Generator(27), _Scores(27)
    audio, target = torch.randn(5, 34, 4), torch.randn(5, 34, 27)
    opts = [_Optim(m, n, log, accelerator.scale) for m, n in ((g, "generator"), (d, "discriminator"))]
    hopmi.train_llm(args, epoch, audio, None, None, target, None, g, d, *opts, accelerator)
    return g


class _Accel:
    """An accelerator that scales the loss, as fp16 training does."""

    def __init__(self, scale, log, **more):
        self.scale, self.log = scale, log
        self.__dict__.update(more)

    def backward(self, loss):
        (loss * self.scale).backward()
        self.log.append(("backward",))

    def unscale_gradients(self, optimizer=None):
        self.log.append(("unscale", optimizer.name))
        optimizer.unscale()


@pytest.mark.parametrize("epoch", [0, 11])
def test_train_llm_clips_unscaled_gradients(epoch, monkeypatch):
    """Under an accelerator that scales the loss, the limit is one on the gradients, not on their scaled form."""
    log = []
    _trace(monkeypatch, log)
    g = _llm(_args(max_grad_norm=0.5), epoch, _Accel(1024.0, log), log)
    assert [e[0] for e in log][-4:] == ["backward", "unscale", "clip", "step"] and log[-3][1] == "generator" and log[-1][1] == "generator"
    assert [id(p) for p in log[-2][1]] == [id(p) for p in g.parameters()] and log[-2][2] == 0.5
    assert [e[0] for e in log].count("clip") == 1 and [e[0] for e in log].count("unscale") == 1
    stepped = log[-1][2]
    # 2^10 scales exactly, so these are the bits of the step without a scale; 16 roundings for a norm of 135 values
    log.clear()
    _llm(_args(max_grad_norm=0.5), epoch, _Accel(1.0, log), log)
    assert abs(_norm(stepped) - 0.5) <= 16 * 2.0 ** -24 and all(torch.equal(a, b) for a, b in zip(stepped, log[-1][2]))


def test_train_llm_clips_only_with_a_limit_and_in_front_of_a_step(monkeypatch):
    """Without a limit the gradients are the optimizer's alone; while an accelerator accumulates, its optimizers do not step."""
    log = []
    _trace(monkeypatch, log)
    for args, more in ((_args(), {}), (_args(max_grad_norm=None), {}), (_args(max_grad_norm=0.5), dict(sync_gradients=False))):
        log.clear()
        _llm(args, 0, _Accel(1024.0, log, **more), log)
        assert [e[0] for e in log] == ["backward", "step"]
    log.clear()
    accel = types.SimpleNamespace(backward=lambda loss: loss.backward(), scale=1.0)          # .backward(loss) is all that is asked for
    _llm(_args(max_grad_norm=0.5), 0, accel, log)
    assert [e[0] for e in log] == ["clip", "step"]


@pytest.mark.parametrize("epoch", [0, 1])
@pytest.mark.parametrize("limit", [None, 0.25, 1e9])
def test_train_iter_gan_clips_the_generators_gradients_in_front_of_its_step(epoch, limit, monkeypatch):
    """backward, clip of exactly the generator's parameters, step; in the discriminator's step nothing is clipped."""
    def run(args):
        torch.manual_seed(4)
        g, d = _Generator(27), _Scores(27)
        audio, poses = torch.randn(5, 34, 4), torch.randn(5, 34, 27)
        hopmi.train_iter_gan(args, epoch, torch.zeros(5, 3), audio, poses, None, g, d, _Optim(g, "generator", log), _Optim(d, "discriminator", log))
        return g

    log = []
    _trace(monkeypatch, log)
    run(_args())
    free = log[:]
    assert [e[:2] for e in free] == [("step", "discriminator")] * epoch + [("step", "generator")] and _norm(free[-1][2]) > 0.5
    log.clear()
    g = run(_args(max_grad_norm=limit))
    assert [e[0] for e in log] == ["step"] * epoch + (["clip"] if limit is not None else []) + ["step"]
    if limit is not None:
        assert [id(p) for p in log[-2][1]] == [id(p) for p in g.parameters()] and log[-2][2] == limit
    if epoch:
        assert all(torch.equal(a, b) for a, b in zip(log[0][2], free[0][2]))
    if limit == 0.25:
        assert abs(_norm(log[-1][2]) - 0.25) <= 16 * 2.0 ** -24                  # (16 roundings; 1e-6 / norm of the formula is below them)
    else:
        assert all(torch.equal(a, b) for a, b in zip(log[-1][2], free[-1][2]))


# -------------------------------------------------------------------------------------------------- which form a product takes
def test_every_form_of_a_product_has_a_size_on_the_device():
    """The lists that the device tests run name all reachable forms, and each size still takes the form that it stands for."""
    import linear_forms as lf
    L = _lib.lib()
    for product, sizes in lf.ALONE.items():
        assert set(sizes) == {(f, s) for f in range(5) for s in (False, True) if not (product == "dw" and f == 1)}, product
        for want, size in sizes.items():
            f, s = lf.form(L, product, size)
            assert (f, s > 1) == want, (product, size)
    assert {k[0] for k in lf.PAIRED} == {2, 3, 4} and len(lf.PAIRED) == 11 and len(lf.SEPARATE) == 4
    for want, size in lf.PAIRED.items():
        pair, f, s, g, t = lf.backward_form(L, size)
        assert pair == 1 and f == g and (f, s > 1, t > 1) == want, size
    for want, size in lf.SEPARATE.items():
        pair, f, s, g, t = lf.backward_form(L, size)
        assert pair == 0 and (s > 1, t > 1) == want, size
        assert (f, s) == lf.form(L, "dx", size) and (g, t) == lf.form(L, "dw", size)
    for blocks, size in lf.FEW.items():
        assert lf.form(L, "y", size) == (-1, 1) and (size[0] + 15) // 16 == blocks


def test_form_queries_refuse_and_agree_with_the_workspaces():
    import ctypes
    import linear_forms as lf
    L = _lib.lib()
    i = ctypes.c_int()
    last = lambda: L.hopmi_last_error().decode()
    for args in ((0, 1, 1, 0), (1, 0, 1, 0), (1, 1, 0, 0), (1, 1, 1, 3), ((1 << 30) + 1, 1, 1, 0)):
        assert L.hopmi_gemm16_form(*args, ctypes.byref(i), ctypes.byref(i)) == -1 and "hopmi_gemm16_form" in last()
    assert L.hopmi_gemm16_form(1, 1, 1, 0, None, ctypes.byref(i)) == -1 and "null" in last()
    p = [ctypes.byref(i)] * 5
    assert L.hopmi_linear16_bwd_form(0, 1, 1, *p) == -1 and L.hopmi_linear16_bwd_form(1, 1, 1, None, *p[1:]) == -1 and "null" in last()
    for product, sizes in lf.ALONE.items():
        for M, K, N in sizes.values():
            a, b, c, layout = {"y": (M, N, K, 0), "dx": (M, K, N, 1), "dw": (N, K, M, 2)}[product]
            s = lf.form(L, product, (M, K, N))[1]
            assert L.hopmi_gemm16_ws_floats(a, b, c, layout) == (s * a * b if s > 1 else 0)
    for M, K, N in [*lf.PAIRED.values(), *lf.SEPARATE.values()]:
        _, _, s, _, t = lf.backward_form(L, (M, K, N))
        assert L.hopmi_linear16_bwd_ws_floats(M, N, K) == (s * M * K if s > 1 else 0) + (t * N * K if t > 1 else 0)


def test_axis_sum_entry_point_refuses():
    import ctypes
    L = _lib.lib()
    one = ctypes.c_void_p(16)                                # (never dereferenced: the checks come first)
    last = lambda: L.hopmi_last_error().decode()
    call = lambda a=one, b=one, it=1, ot=1, outer=1, R=100000, inner=768, ws=one: L.hopmi_axis_sum(a, it, b, ot, outer, R, inner, ws, None)
    assert call(a=None) == -1 and "null" in last()
    assert call(b=None) == -1 and "null" in last()
    for kw in (dict(outer=0), dict(R=0), dict(inner=0), dict(outer=-1), dict(R=1 << 41), dict(outer=1 << 30, R=1 << 30), dict(outer=1 << 20, R=1 << 20, inner=2)):
        assert call(**kw) == -1 and "2^40" in last(), kw
        assert L.hopmi_axis_sum_ws_floats(kw.get("outer", 1), kw.get("R", 5), kw.get("inner", 768)) == 0
    for kw in (dict(it=3), dict(ot=-1), dict(it=1, ot=2)):
        assert call(**kw) == -1 and "dtype" in last(), kw
    assert L.hopmi_axis_sum_ws_floats(1, 100000, 768) > 0 and call(ws=None) == -1 and "workspace" in last()
    assert L.hopmi_axis_sum_ws_floats(1000, 100, 768) == 0 and L.hopmi_axis_sum_ws_floats(1, 1, 1) == 0
    # groups of whole rows: a workspace of at most 1024 partial rows per outer index, never more than the input
    for outer, R, inner in ((1, 5, 64), (1, 33, 64), (1, 1 << 30, 1), (7, 4097, 3), (1, 2, 1 << 20), (1 << 20, 1 << 10, 1), (3, 1 << 20, 65)):
        n = L.hopmi_axis_sum_ws_floats(outer, R, inner)
        assert n % (outer * inner) == 0 and n <= 1024 * outer * inner and n <= outer * R * inner
