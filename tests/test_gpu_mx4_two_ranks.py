"""Two data-parallel ranks on one GPU training from 4-bit stores of their own with a teacher: the step in its parts, its all-reduce,
accumulation and loss scale, against an in-process simulation of the two ranks with the gradients summed by hand.  Collectives go through
host memory (gloo takes CPU tensors here)."""
import os
import sys
from argparse import Namespace

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
N, D, Q, C, B, IMAGES = 21, 256, 8, 30, 12, 40
LRS = [0.05, 0.3, 0.2]


def _engine(world, accum, scaler, overlap):
    from efficient_probing_amd import probe_heads
    from efficient_probing_amd.engine import ProbeHeadEngine
    from efficient_probing_amd.util.misc import NativeScalerWithGradNormCount
    torch.manual_seed(0)
    m = torch.nn.Module()
    m.head = torch.nn.Linear(D, C)
    probe_heads.build_probe_head(m, Namespace(cls_features="ep", ep_queries=Q, d_out=1, nb_classes=C))
    eng = ProbeHeadEngine(m.head.to("cuda:0").train(), optimizer="lars", weight_decay=1e-3, accum_iter=accum, overlap_comm=overlap)
    eng.world = world
    if scaler:
        eng.attach_scaler(NativeScalerWithGradNormCount())
    return eng


def _store(rank):
    """A rank's own images, lengths and teacher rows; batches through an index."""
    from efficient_probing_amd import distill, mx4
    g = torch.Generator().manual_seed(100 + rank)
    lengths = torch.randint(1, N + 1, (IMAGES,), generator=g, dtype=torch.int32).to("cuda:0")
    cache = mx4.quantize_tokens(torch.randn(IMAGES, N, D, generator=g).to("cuda:0"), lengths=lengths)
    crit = distill.TopKDistillation(*distill.teacher_topk(torch.randn(IMAGES, C, generator=g).to("cuda:0"), 5, 2.0), temperature=2.0, alpha=0.6)
    return cache, torch.randint(0, C, (IMAGES,), generator=g).to("cuda:0"), crit, g


def _batch(g, labels):
    idx = torch.randperm(IMAGES, generator=g)[:B].to(torch.int32).to("cuda:0")
    return idx, labels[idx.long()]


def _worker(rank, world, port, out_dir, accum, scaler, teacher, overlap):
    sys.path.insert(0, ROOT)
    import torch.distributed as dist
    os.environ["MASTER_ADDR"] = "127.0.0.1"; os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.cuda.set_device(0)

    def through_host(collective):
        def call(t, *a, async_op=False, **kw):
            assert not async_op
            host = t.cpu()
            collective(host, *a, **kw)
            t.copy_(host)
        return call
    dist.all_reduce, dist.broadcast = through_host(dist.all_reduce), through_host(dist.broadcast)
    eng = _engine(world, accum, scaler, overlap)
    cache, labels, crit, g = _store(rank)
    for lr in LRS:
        for _ in range(accum):
            idx, tgt = _batch(g, labels)
            eng.train_step(cache, tgt, lr=lr, image_index=idx, criterion=crit if teacher else None)
    eng.flush()
    eng.sync_buffers()
    torch.cuda.synchronize()
    torch.save({"p": eng.flat_p.cpu(), "mu": eng.state[0].cpu(), "rm": eng.bn.running_mean.cpu(), "stats": eng.read_stats()}, os.path.join(out_dir, f"rank{rank}.pt"))
    dist.destroy_process_group()


@pytest.mark.parametrize("accum,scaler,teacher,overlap", [(1, False, True, None), (2, False, True, None), (1, True, True, None), (1, False, False, None), (1, False, True, True)])
def test_two_ranks_equal_simulation(tmp_path, accum, scaler, teacher, overlap):
    import torch.multiprocessing as mp
    world, port = 2, 29150 + (os.getpid() % 200)
    mp.spawn(_worker, args=(world, port, str(tmp_path), accum, scaler, teacher, overlap), nprocs=world, join=True)
    got = [torch.load(os.path.join(tmp_path, f"rank{r}.pt")) for r in range(world)]
    assert torch.equal(got[0]["p"], got[1]["p"]) and torch.equal(got[0]["mu"], got[1]["mu"]) and torch.equal(got[0]["rm"], got[1]["rm"])
    reps, stores = [_engine(world, accum, scaler, False) for _ in range(world)], [_store(r) for r in range(world)]
    start = reps[0].flat_p.clone()
    for lr in LRS:
        for _ in range(accum):
            for e, (cache, labels, crit, g) in zip(reps, stores):
                idx, tgt = _batch(g, labels)
                e.forward_backward_parts(cache, tgt, idx, crit if teacher else None)
        total = reps[0].flat_g + reps[1].flat_g
        for e in reps:
            e.flat_g.copy_(total)
            e.optimizer_step(lr)
    assert not torch.equal(reps[0].flat_p, start)
    assert torch.equal(reps[0].flat_p, reps[1].flat_p) and torch.equal(got[0]["p"], reps[0].flat_p.cpu())
    for r, e in enumerate(reps):
        assert got[r]["stats"] == e.read_stats()
