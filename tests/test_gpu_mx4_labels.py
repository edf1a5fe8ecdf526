"""Distillation with images that carry no label: they train from their teacher alone and are no hit of the accuracy counts."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _head(D, C, favourite):
    """An EP head whose every prediction is ``favourite``."""
    from argparse import Namespace
    from efficient_probing_amd import probe_heads
    torch.manual_seed(0)
    m = torch.nn.Module()
    m.head = torch.nn.Linear(D, C)
    probe_heads.build_probe_head(m, Namespace(cls_features="ep", ep_queries=4, d_out=1, nb_classes=C))
    with torch.no_grad():
        m.head[2].bias[favourite] += 100.0
    return m.to(DEV).head.train()


@pytest.mark.parametrize("alpha", [1.0, 0.5])
@pytest.mark.parametrize("cached", [False, True])
def test_unlabelled_images_are_no_hit(alpha, cached):
    from efficient_probing_amd import distill, mx4
    from efficient_probing_amd.engine import ProbeHeadEngine
    B, N, D, C = 16, 9, 128, 11
    g = torch.Generator().manual_seed(1)
    x = torch.randn(B, N, D, generator=g).to(DEV)
    values, index, tail = distill.teacher_topk(torch.randn(B, C, generator=g).to(DEV), 4, 2.0)
    crit = distill.TopKDistillation(values, index, tail, temperature=2.0, alpha=alpha)
    tgt = torch.tensor([0, 0, 3, -1, -100, 0, -1, 7, 0, -2, -1, -1, 5, -100, 0, -1], device=DEV)
    eng = ProbeHeadEngine(_head(D, C, 0), optimizer="sgd", lr=0.0)
    eng.forward_backward_parts(mx4.quantize_tokens(x) if cached else x, tgt, None, crit)
    loss, top1, top5, bad = eng.read_stats()
    logits = eng.last_train_logits()
    assert bool((logits.argmax(1) == 0).all())
    five = (logits.topk(5, 1).indices == tgt[:, None]).any(1)
    assert (top1, top5, bad) == (5.0, float(five.sum()), 0.0)


def test_a_label_out_of_range_is_no_hit():
    from efficient_probing_amd import functional as F_
    z = torch.zeros(6, 5, device=DEV)
    z[:, 0] = 3.0
    rows, _, stats = F_.cross_entropy(z, torch.tensor([0, -1, 5, 1, -100, 2 ** 40], device=DEV))
    assert stats[1:].tolist() == [1.0, 2.0, 4.0]
    assert rows[:, 1].tolist() == [1, 0, 0, 0, 0, 0] and rows[:, 3].tolist() == [0, 1, 1, 0, 1, 1]
