"""Tests.  Importing the package (pytest does, and so does every rank that a test spawns) gives gloo host memory only: its
collectives on device tensors can hang where ranks share a GPU, and some tests hand theirs to torch.distributed directly."""
import torch.distributed as dist


def host_only(reduce):
    """`reduce` (dist.all_reduce), but under gloo a device tensor goes through host memory, with synchronous copies."""
    def all_reduce(tensor, op=dist.ReduceOp.SUM, group=None, async_op=False):
        if not (tensor.is_cuda and dist.get_backend(group) == "gloo"):
            return reduce(tensor, op=op, group=group, async_op=async_op)
        if async_op:
            raise RuntimeError("a device tensor under gloo: use parallel.all_reduce")
        host = tensor.detach().cpu()
        reduce(host, op=op, group=group)
        tensor.data.copy_(host)
    all_reduce.host_only = True
    return all_reduce


if dist.is_available() and not getattr(dist.all_reduce, "host_only", False):
    dist.all_reduce = host_only(dist.all_reduce)
