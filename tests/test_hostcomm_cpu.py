"""hostcomm without a GPU: which collectives go through host memory, and that a staged sum reaches its tensor once."""
import os
import sys
from types import SimpleNamespace

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import _gloo_host

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


def _worker(rank, store, q):
    sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
    import _parity  # noqa: F401 -- what the GPU tests' workers import before they exchange anything
    dist.init_process_group("gloo", init_method=f"file://{store}", rank=rank, world_size=2)
    hostcomm.staged = lambda t, group: t.numel() > 2               # stands for a device tensor
    seen, wrapped = [], sys.modules["_gloo_host"]
    wrapped.plain = lambda parts, t, group=None, async_op=False, plain=wrapped.plain: (seen.append(t.numel()), plain(parts, t, group=group, async_op=async_op))[1]
    got = []
    for n in (2, 5):
        t = torch.arange(float(n)) + 10 * rank
        parts = [torch.full((n,), -1.) for _ in range(2)]
        dist.all_gather(parts, t)
        got.append([p.tolist() for p in parts])
    q.put((rank, got, seen, dist.all_gather is wrapped.all_gather))
    dist.destroy_process_group()


def test_workers_gather_through_host_memory(tmp_path):
    assert dist.all_gather is _gloo_host.plain                     # not in a program of its own
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    ps = [ctx.Process(target=_worker, args=(r, str(tmp_path / "store"), q)) for r in range(2)]
    for p in ps:
        p.start()
    res = sorted(q.get(timeout=120) for _ in ps)
    for p in ps:
        p.join(60)
    for rank, got, seen, wrapped in res:
        assert wrapped and seen == [2, 5]
        assert got == [[[0., 1.], [10., 11.]], [[float(i) for i in range(5)], [10. + i for i in range(5)]]]
