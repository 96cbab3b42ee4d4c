"""gloo gets host memory only, also from tests that call torch.distributed themselves, in this process and in spawned ranks."""
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import tests


class _Device(torch.Tensor):
    """A host tensor that says it is a device's."""
    is_cuda = property(lambda self: True)

    def detach(self):
        return self

    def cpu(self):
        return self.as_subclass(torch.Tensor).clone()


def test_device_tensors_are_staged_and_host_tensors_are_not(tmp_path):
    dist.init_process_group("gloo", init_method="file://%s" % (tmp_path / "store"), rank=0, world_size=1)
    try:
        handed = []
        reduce = tests.host_only(lambda t, op, group, async_op=False: (handed.append(t), t.mul_(2), op)[-1])
        t = torch.arange(3.0)
        assert reduce(t, op=dist.ReduceOp.MAX) == dist.ReduceOp.MAX and handed.pop() is t and t.tolist() == [0, 2, 4]
        d = torch.arange(3.0).as_subclass(_Device)
        reduce(d)
        assert not handed[-1].is_cuda and handed.pop().data_ptr() != d.data_ptr() and d.tolist() == [0, 2, 4]
        with pytest.raises(RuntimeError):
            reduce(d, async_op=True)
        assert not handed
    finally:
        dist.destroy_process_group()


def _rank(q):
    q.put(getattr(dist.all_reduce, "host_only", False))


def test_spawned_ranks_have_it_too():
    assert dist.all_reduce.host_only
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    p = ctx.Process(target=_rank, args=(q,))
    p.start()
    assert q.get(timeout=120) is True
    p.join(60)
    assert p.exitcode == 0
