"""CPU: what the trainable block's operators refuse (layer_norm, linear_act, GradClip / clip_grad_norm_), in Python and at the C entry
points.  Every check comes before any launch: nothing here touches a device."""
import ctypes

import pytest
import torch

import hopmi
from hopmi import _lib

ops = hopmi.ops
ONE = ctypes.c_void_p(16)                    # (never dereferenced: the checks come first)


def _last():
    return _lib.lib().hopmi_last_error().decode()


def test_host_tensors_and_bad_arguments_are_refused():
    x = torch.zeros(4, 8)
    for call in (lambda: ops.layer_norm(x), lambda: ops.linear_act(x.bfloat16(), x.bfloat16()), lambda: ops.GradClip([x])):
        with pytest.raises(_lib.HopmiError, match="no CPU fallback"):
            call()
    with pytest.raises(_lib.HopmiError, match="type"):
        ops.layer_norm(x.double())
    with pytest.raises(_lib.HopmiError, match="shape"):
        ops.layer_norm(torch.zeros(()))
    with pytest.raises(_lib.HopmiError, match="activation"):
        ops.linear_act(x, x, activation="tanh")
    with pytest.raises(_lib.HopmiError, match="empty list"):
        ops.GradClip([])
    with pytest.raises(_lib.HopmiError, match="one axis"):
        ops.LayerNorm((4, 8))
    assert float(ops.clip_grad_norm_([], 1.0)) == 0.0
    assert float(ops.clip_grad_norm_([torch.nn.Parameter(x)], 1.0)) == 0.0
    assert list(ops.LayerNorm(8).state_dict()) == list(torch.nn.LayerNorm(8).state_dict())


def test_layernorm_entry_points_refuse():
    L = _lib.lib()
    args = lambda dt=0, wdt=0, M=4, D=8, ld=8, eps=1e-5, x=ONE: L.hopmi_layernorm_fwd(x, ld, ONE, ONE, wdt, ONE, None, None, M, D, eps, dt, None)
    for bad, word in ((args(dt=3), "dtype"), (args(dt=1, wdt=2), "dtype"), (args(M=0), "sizes"), (args(D=0), "sizes"), (args(ld=7), "sizes")):
        assert bad == -1
    assert args(eps=-1.0) == -1 and "eps" in _last()
    assert args(x=None) == -1 and "null" in _last()
    assert L.hopmi_layernorm_fwd(ONE, 8, ONE, ONE, 0, ONE, ONE, None, 4, 8, 1e-5, 0, None) == -1            # one of the statistics
    assert L.hopmi_layernorm_bwd(ONE, 8, ONE, ONE, ONE, ONE, 0, ONE, ONE, ONE, None, 4, 8, 0, None) == -1 and "null" in _last()
    assert L.hopmi_layernorm_bwd(ONE, 8, ONE, ONE, ONE, ONE, 0, None, None, None, None, 4, 8, 0, None) == 0  # nothing wanted, nothing done
    assert L.hopmi_layernorm_bwd_ws_floats(0, 8, 0) == 0 and L.hopmi_layernorm_bwd_ws_floats(4, 8, 0) == 16


def test_gemm16_entry_points_refuse():
    L = _lib.lib()

    def call(A=ONE, lda=64, B=ONE, ldb=64, layout=0, C=ONE, ldc=128, act=0, M=128, N=128, K=64, dt=1, ws=ONE, res=None, ldr=0):
        return L.hopmi_gemm16(A, lda, B, ldb, layout, C, ldc, None, res, ldr, None, 0, act, M, N, K, dt, ws, None)

    assert call(A=None) == -1 and "null" in _last()
    for kw in (dict(M=0), dict(N=0), dict(K=0), dict(layout=3), dict(act=4)):
        assert call(**kw) == -1
    assert call(dt=0) == -1 and "dtype" in _last()
    for kw in (dict(lda=63), dict(ldb=56), dict(ldc=127), dict(res=ONE, ldr=100)):
        assert call(**kw) == -1 and "stride" in _last(), kw
    assert call(lda=1 << 23) == -1 and "2^22" in _last()
    assert call(M=(1 << 31) - 1, N=(1 << 31) - 1, ldc=1 << 31) == -1 and "more tiles" in _last()
    for kw in (dict(A=ctypes.c_void_p(18)), dict(lda=68), dict(lda=62, K=62), dict(ldb=128, ldc=128, N=122, lda=60, K=60, layout=1), dict(B=ctypes.c_void_p(24))):
        assert call(**kw) == -1 and "16 bytes" in _last(), kw
    assert L.hopmi_gemm16_ws_floats(128, 128, 4096, 0) > 0
    assert call(K=4096, lda=4096, ldb=4096, ws=None) == -1 and "workspace" in _last()
    assert L.hopmi_gemm16_ws_floats(16, 128, 768, 0) == 0 and L.hopmi_gemm16_ws_floats(0, 1, 1, 0) == 0
    assert L.hopmi_gemm16_direct(ONE, 64, 64) == 1 and L.hopmi_gemm16_direct(ONE, 1 << 23, 64) == 0 and L.hopmi_gemm16_direct(ONE, 64, 60) == 0 and L.hopmi_gemm16_direct(ctypes.c_void_p(8), 64, 64) == 0
    assert L.hopmi_pad16(ONE, 5, ONE, 12, 4, 5, None) == -1 and L.hopmi_pad16(ONE, 5, ctypes.c_void_p(8), 8, 4, 5, None) == -1
    for kw in (dict(act=2, z=None), dict(ldz=12), dict(ws=None), dict(ldd=12), dict(dt=0)):
        a = dict(act=1, z=ONE, ldz=16, ws=ONE, ldd=16, dt=1)
        a.update(kw)
        assert L.hopmi_act_bwd16(ONE, 13, a["z"], a["ldz"], ONE, a["ldd"], ONE, a["ws"], a["act"], 4, 13, a["dt"], None) == -1, kw


def test_grad_clip_entry_point_refuses():
    L = _lib.lib()
    ptr, n, dt = (ctypes.c_void_p * 1)(16), (ctypes.c_longlong * 1)(4), (ctypes.c_int * 1)(0)
    assert L.hopmi_grad_clip(ptr, None, n, dt, -1, 1.0, ONE, ONE, None) == -1
    assert L.hopmi_grad_clip(None, None, n, dt, 1, 1.0, ONE, ONE, None) == -1
    assert L.hopmi_grad_clip(ptr, None, n, dt, 1, 1.0, None, ONE, None) == -1 and "null" in _last()
    assert L.hopmi_grad_clip(ptr, None, n, dt, 1, -1.0, ONE, ONE, None) == -1 and "max_norm" in _last()
    assert L.hopmi_grad_clip(ptr, None, n, dt, 1, float("nan"), ONE, ONE, None) == -1
    for bn, bdt, bp in ((-1, 0, 16), (4, 3, 16), (4, 0, None)):
        assert L.hopmi_grad_clip((ctypes.c_void_p * 1)(bp), None, (ctypes.c_longlong * 1)(bn), (ctypes.c_int * 1)(bdt), 1, 1.0, ONE, ONE, None) == -1
        assert "tensor 0" in _last()
    many = 250 * 129
    assert L.hopmi_grad_clip((ctypes.c_void_p * many)(*[16] * many), None, (ctypes.c_longlong * many)(*[1] * many),
                             (ctypes.c_int * many)(), many, 1.0, ONE, ONE, None) == -1 and "more than one call" in _last()


def test_recorded_step_over_ranks_refuses_max_grad_norm(tmp_path):
    """The recorded step shards the mapping layer's gradient over the ranks: no rank has the norm."""
    import types

    import torch.distributed as dist
    mod = torch.nn.Linear(2, 2)
    args = types.SimpleNamespace(max_grad_norm=1.0)
    assert not hopmi.GraphedTrainStep(args, mod, mod, None, None).exchange            # one rank: accepted
    if dist.is_initialized():
        pytest.skip("a process group is up in this process")
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        with pytest.raises(_lib.HopmiError, match="max_grad_norm"):
            hopmi.GraphedTrainStep(args, mod, mod, None, None, force_exchange=True)
        assert hopmi.GraphedTrainStep(types.SimpleNamespace(), mod, mod, None, None, force_exchange=True).exchange
    finally:
        dist.destroy_process_group()


def test_sizes_that_indices_do_not_count_are_refused():
    L = _lib.lib()
    big, most = (1 << 31) - 1, 1 << 30
    assert L.hopmi_layernorm_fwd(ONE, big, ONE, ONE, 0, ONE, None, None, 4, most, 1e-5, 0, None) == -1 and "sizes" in _last()
    assert L.hopmi_layernorm_bwd(ONE, big, ONE, ONE, ONE, ONE, 0, ONE, ONE, ONE, ONE, 4, most, 0, None) == -1 and "sizes" in _last()
    assert L.hopmi_layernorm_bwd_ws_floats(4, most, 0) == 0 and L.hopmi_layernorm_bwd_ws_floats(4, 1 << 29, 0) == 1 << 32
    gemm = lambda M, N, K, layout: L.hopmi_gemm16(ONE, 1 << 32, ONE, 1 << 32, layout, ONE, 1 << 32, None, None, 0, None, 0, 0, M, N, K, 1, ONE, None)
    for layout in range(3):
        for side in ((most + 1, 8, 8), (8, most + 1, 8), (8, 8, most + 1), (4, 8, big)):
            assert gemm(*side, layout) == -1 and "2^30" in _last(), (side, layout)
            assert L.hopmi_gemm16_ws_floats(*side, layout) == 0
    assert L.hopmi_act_bwd16(ONE, 1 << 32, ONE, 1 << 32, ONE, 1 << 32, ONE, ONE, 1, 4, most + 1, 1, None) == -1
    assert L.hopmi_act_bwd16_ws_floats(4, most + 1) == 0


def test_tangents_and_pending_negations_are_refused():
    """The kernels read memory: a forward-mode tangent would be lost, a pending negation not applied."""
    import torch.autograd.forward_ad as fwad
    x, w = torch.zeros(4, 8), torch.zeros(8, 8)
    with fwad.dual_level():
        d = fwad.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.layer_norm(d), lambda: ops.layer_norm(x, d[0]), lambda: ops.linear_act(d, w), lambda: ops.linear_act(x, w, None, d)):
            with pytest.raises(_lib.HopmiError, match="forward-mode"):
                call()
    n = torch.complex(x, x).conj().imag
    assert n.is_neg()
    for call in (lambda: ops.layer_norm(n), lambda: ops.linear_act(n, w), lambda: ops.linear_act(x, w, n[0])):
        with pytest.raises(_lib.HopmiError, match="negation"):
            call()


def test_linear16_bwd_entry_point_refuses():
    L = _lib.lib()

    def call(dz=ONE, lddz=64, w=ONE, ldw=72, x=ONE, ldx=72, dx=ONE, dw=ONE, part=ONE, db=ONE, M=100, N=64, K=72, dt=1, ws=ONE):
        return L.hopmi_linear16_bwd(dz, lddz, w, ldw, x, ldx, dx, dw, part, db, M, N, K, dt, ws, None)

    for kw in (dict(dz=None), dict(w=None), dict(x=None), dict(dx=None), dict(dw=None), dict(part=None)):
        assert call(**kw) == -1 and "null" in _last(), kw
    for kw in (dict(M=0), dict(N=0), dict(K=0), dict(dt=0), dict(M=(1 << 30) + 1)):
        assert call(**kw) == -1 and "M=" in _last(), kw
    odd = ctypes.c_void_p(24)
    for kw in (dict(dz=odd), dict(w=odd), dict(x=odd), dict(lddz=56), dict(ldw=76), dict(ldx=64), dict(lddz=60, N=60), dict(K=73), dict(ldx=1 << 23)):
        assert call(**kw) == -1 and "16 bytes" in _last(), kw
    assert L.hopmi_linear16_bwd_ws_floats(16000, 40, 40) > 0 and L.hopmi_linear16_bwd_ws_floats(65, 40, 72) == 0
    assert L.hopmi_linear16_bwd_ws_floats(0, 40, 72) == 0
    assert call(M=16000, N=40, K=40, ws=None) == -1 and "workspace" in _last()
    two = lambda **kw: L.hopmi_pad16_two(ONE, 5, ONE, kw.get("ldp", 8), 4, 5, ONE, 5, kw.get("dst2", ONE), 8, kw.get("M2", 4), 5, None)
    assert two(ldp=12) == -1 and two(dst2=ctypes.c_void_p(8)) == -1 and two(M2=0) == -1 and "pad16" in _last()
    assert call(M=1 << 30, N=1 << 22, K=1 << 22, lddz=1 << 22, ldw=1 << 22, ldx=1 << 22) == -1 and "more tiles" in _last()
