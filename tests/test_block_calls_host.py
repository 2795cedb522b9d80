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
