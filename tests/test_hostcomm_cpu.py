"""hostcomm without a GPU: which collectives go through host memory, and that a staged sum reaches its tensor once."""
from types import SimpleNamespace

import pytest
import torch
import torch.distributed as dist

from unimp_amd import hostcomm

# a group's name (dist.get_backend) and its backend for every device type (dist.get_backend_config)
GROUPS = {"gloo": "cpu:gloo,cuda:gloo", "nccl": "cuda:nccl", "undefined": "cpu:gloo,cuda:nccl", "cpu:gloo,cuda:nccl": "cpu:gloo,cuda:nccl", "cuda:nccl": "cuda:nccl",
          "cuda:gloo": "cuda:gloo", "cpu:gloo": "cpu:gloo"}


@pytest.mark.parametrize("name", GROUPS)
def test_only_gloos_own_device_path_is_staged(monkeypatch, name):
    """a group without a named backend, or with one per device type, moves device tensors over RCCL: they are not copied to the host"""
    monkeypatch.setattr(dist, "get_backend", lambda group=None: name)
    monkeypatch.setattr(dist, "get_backend_config", lambda group=None: GROUPS[name])
    device = SimpleNamespace(is_cuda=True)
    assert hostcomm.staged(device, None) is ("cuda:gloo" in GROUPS[name])
    assert hostcomm.staged(torch.zeros(1), None) is False


def test_config_of_a_real_group(tmp_path):
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        assert hostcomm.staged(SimpleNamespace(is_cuda=True), None) and hostcomm.staged(SimpleNamespace(is_cuda=True), dist.group.WORLD)
        t = torch.arange(4.)
        hostcomm.all_reduce(t, dist.ReduceOp.SUM, None)
        out = torch.zeros(4)
        hostcomm.all_gather_cat(out, t, 1, None)
        assert torch.equal(out, torch.arange(4.))
    finally:
        dist.destroy_process_group()


def test_a_second_wait_changes_nothing(monkeypatch):
    """the sum is copied over its tensor once: what was written there since stays"""
    monkeypatch.setattr(dist, "all_reduce", lambda t, op, group, async_op: SimpleNamespace(wait=lambda: None))
    t = torch.ones(3)
    h = hostcomm._Staged(t, dist.ReduceOp.SUM, None)
    h.host = torch.full((3,), 2.)                                   # the sum (a host copy of a host tensor is the tensor itself)
    h.wait()
    assert torch.equal(t, torch.full((3,), 2.))
    t.fill_(5.)                                                     # the next step's gradients
    h.wait()
    assert torch.equal(t, torch.full((3,), 5.))
