"""Collectives on device tensors whose group hands them to gloo (CPU runs' backend, also of several ranks that share one GPU): staged through host memory with synchronous copies,
because gloo's own device path works on streams of another priority and has hung where several ranks shared a card.  Every other backend takes the tensor itself."""
import torch
import torch.distributed as dist


def staged(t, group):
    """does a collective of ``group`` on ``t`` go through host memory?  Decided by the backend that the group has for the tensor's device type: a group's name does not tell it (made
    without a backend it is "undefined", with one per device type "cpu:gloo,cuda:nccl"; both take device tensors over RCCL)"""
    return t.is_cuda and "cuda:gloo" in str(dist.get_backend_config(group)).split(",")


class _Staged:
    """handle of an asynchronous all-reduce of a host copy; the sum reaches the device tensor in the first wait()"""

    def __init__(self, t, op, group):
        self.t, self.host = t, t.to("cpu")                    # synchronous: every kernel that writes t has finished
        self.work = dist.all_reduce(self.host, op=op, group=group, async_op=True)

    def wait(self):
        self.work.wait()
        if self.t is not None:
            self.t.copy_(self.host)
            self.t = None


def all_reduce(t, op, group, async_op=False):
    """in place; returns a handle if async_op"""
    if not staged(t, group):
        return dist.all_reduce(t, op=op, group=group, async_op=async_op)
    h = _Staged(t, op, group)
    if async_op:
        return h
    h.wait()


def all_gather_cat(out, mine, world, group):
    """out [world * n] = the ranks' ``mine`` [n] in rank order"""
    src = mine.to("cpu") if staged(mine, group) else mine.contiguous()
    parts = [torch.empty_like(src) for _ in range(world)]
    dist.all_gather(parts, src, group=group)
    out.copy_(torch.cat(parts))
