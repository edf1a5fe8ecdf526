"""The distillation's gradient class by class: most of a long row are classes that the teacher does not list, each with a share far below
the largest component, and each has to be right relative to its own terms.

Bound of a component (u = 2^-24), on the sizes of the terms that it is a sum of (oracle ``sizes``): an exponential is off by 4 u (the
instruction, its sum's and its quotient's rounding) plus 4 u times its argument (the difference's rounding, the factor log2(e) / T and the
product's), and arguments that count in a sum are log C <= 14 in the mean: 64 u for a sum; the teacher's side likewise with arguments of
the size of its logits over T.  r = 192 u + 8 u (|argument| + teacher's).  Then one rounding to the logits' type (half a step), half of
its smallest subnormal, and 2^-126 per term, below which an exponential is zero."""
import numpy as np
import pytest
import torch

from oracle import distill_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def _teacher(R, C, K, seed):
    rng = np.random.default_rng(seed)
    start, step = rng.integers(0, C, (R, 1)), max(1, C // K)
    idx = np.stack([(start[r] + step * rng.permutation(K)) % C for r in range(R)]).astype(np.int32)
    return (6 + 3 * rng.standard_normal((R, K))).astype(np.float32), idx, (4 + rng.standard_normal(R)).astype(np.float32)


def _check(z, val, idx, tgt, tail, T, alpha, gs):
    from efficient_probing_amd import distill
    B, C = z.shape
    dev = lambda a: None if a is None else torch.as_tensor(a, device=DEV)
    zf = z.double().cpu().numpy()
    want = O.distill(zf, val, idx, tgt, tail, T, alpha)[1] * (gs / B)
    mag, far = O.sizes(zf, val, idx, tgt, tail, T, alpha)
    _, grad = distill.topk_distillation(z, dev(val), dev(idx), dev(tgt), teacher_tail=dev(tail), temperature=T, alpha=alpha, grad_scale=gs)
    t = np.abs(val).max() / T + (0.0 if tail is None else np.abs(tail).max()) + 14.0
    lim = (gs / B) * (mag * (192 * U + 8 * U * (far + t)) + 4 * T * 2.0 ** -126) + np.abs(want) * torch.finfo(z.dtype).eps / 2 + TINY[z.dtype]
    err = np.abs(grad.double().cpu().numpy() - want)
    assert (err <= lim).all(), (float((err / lim).max()), np.unravel_index((err / lim).argmax(), err.shape), float((err > lim).mean()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,C,K", [(3, 2, 1), (5, 63, 5), (4, 1000, 32), (3, 4099, 100), (2, 10000, 16), (2, 21841, 64), (1, 32768, 64), (2, 65537, 256),
                                   (2, 131071, 128), (1, 1 << 20, 1024)])
@pytest.mark.parametrize("mode", ["soft", "soft+label", "tail", "tail+label"])
def test_every_class_by_its_own_terms(B, C, K, dtype, mode):
    """(the loss scale keeps the shares of unlisted classes within fp16's range)"""
    z = (2 * torch.randn(B, C, generator=torch.Generator().manual_seed(C))).to(dtype).to(DEV)
    val, idx, tail = _teacher(B, C, K, C + K)
    label = "label" in mode
    tgt = np.random.default_rng(B + C).integers(0, C, B) if label else None
    _check(z, val, idx, tgt, tail if "tail" in mode else None, 2.0 if label else 1.0, 0.4 if label else 1.0, 4096.0)


@pytest.mark.parametrize("C", [50, 3000, 21841, 40001])
@pytest.mark.parametrize("gap", [30.0, 45.0, 60.0, 66.0, 75.0, 200.0])
def test_shares_far_below_the_list(C, gap):
    """The classes behind the list from near its logits to beyond fp32's range below them, with a spread of their own."""
    B, K = 3, 8
    val, idx, tail = _teacher(B, C, K, C)
    z = 3 * torch.randn(B, C, generator=torch.Generator().manual_seed(C))
    z.scatter_add_(1, torch.as_tensor(idx, dtype=torch.long), torch.full((B, K), gap))
    _check(z.to(DEV), val, idx, None, tail, 1.0, 1.0, 1.0)
    _check(z.to(DEV), val, idx, np.array([0, int(idx[1, 0]), -1]), tail, 1.0, 0.5, 1.0)


@pytest.mark.parametrize("C", [40, 5000, 40001])
@pytest.mark.parametrize("tail_on", [False, True])
def test_without_weight_the_teacher_does_not_count(C, tail_on):
    """alpha = 0 is the cross-entropy alone, also where the distillation term would be infinite or not a number: the student gives a
    listed class no mass, nothing is left for the tail, the teacher's logits are NaN."""
    from efficient_probing_amd import distill
    B, K = 5, 6
    val, idx, tail = _teacher(B, C, K, C)
    z = torch.randn(B, C, generator=torch.Generator().manual_seed(C))
    z[0, int(idx[0, 0])] = -np.inf
    z[1] = torch.where(torch.zeros(C, dtype=torch.bool).scatter(0, torch.as_tensor(idx[1], dtype=torch.long), True), z[1], torch.tensor(-np.inf))
    val[2, 1], val[3, 0] = np.nan, np.inf
    tail[4] = np.nan
    tgt = torch.tensor([int(idx[b, 3]) for b in range(B)])
    ref = z.double().requires_grad_(True)
    want = torch.nn.functional.cross_entropy(ref, tgt, reduction="none")
    want.sum().backward()
    dev = lambda a: torch.as_tensor(a, device=DEV)
    loss, grad = distill.topk_distillation(z.to(DEV), dev(val), dev(idx), tgt.to(DEV), teacher_tail=dev(tail) if tail_on else None, temperature=2.0, alpha=0.0, grad_scale=float(B))
    assert (loss.double().cpu() - want.detach()).abs().max() <= 192 * U * 20
    one = torch.nn.functional.one_hot(tgt, C)
    assert ((grad.double().cpu() - ref.grad).abs() <= 320 * U * (ref.grad.abs() + 2 * one) + 2.0 ** -126).all()


def test_a_teacher_that_requires_gradients():
    """The teacher's logits of a model that trains elsewhere: it takes no gradient, the student does; without a student that trains the loss
    is a constant."""
    from efficient_probing_amd import distill
    B, C, K = 4, 50, 6
    val, idx, tail = _teacher(B, C, K, 1)
    v, t = torch.as_tensor(val, device=DEV).requires_grad_(), torch.as_tensor(tail, device=DEV).requires_grad_()
    i, z = torch.as_tensor(idx, device=DEV), torch.randn(B, C, device=DEV)
    assert not distill.distillation_loss(z, v, i, teacher_tail=t).requires_grad
    q = z.clone().requires_grad_()
    loss = distill.distillation_loss(q, v * 1.0, i, teacher_tail=t * 1.0)
    loss.backward()
    rows, grad = distill.topk_distillation(z, v, i, teacher_tail=t)
    assert v.grad is None and t.grad is None and torch.equal(q.grad, grad) and not rows.requires_grad and not grad.requires_grad


def test_captured_means_of_growing_batches():
    """One graph after another, up to batches whose mean would take several workgroups: replays follow the logits, with eager work between."""
    from efficient_probing_amd import distill
    for B in (1000, 20000, 100000, 300000, 2000000):
        g = torch.Generator(device=DEV).manual_seed(1)
        z, v = torch.randn(B, 4, device=DEV, generator=g), torch.randn(B, 2, device=DEV, generator=g)
        i = torch.randint(0, 4, (B, 2), device=DEV, generator=g, dtype=torch.int32)
        zs = z.clone()
        distill.distillation_loss(zs, v, i)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = distill.distillation_loss(zs, v, i)
        for k in range(6):
            zs.copy_(z * (k + 1))
            want = distill.distillation_loss(zs, v, i)
            torch.randn(1000000, device=DEV).sum().item()
            graph.replay()
            torch.cuda.synchronize()
            assert float(out) == float(want), (B, k)


def test_mean_of_many_rows():
    from efficient_probing_amd import distill
    for n in (1, 65536, 65537, 66000, 300001, 2 ** 21 + 3):
        rows = torch.rand(n, generator=torch.Generator().manual_seed(n)) + 0.5
        assert abs(float(distill.mean_rows(rows.to(DEV))) - float(rows.double().mean())) <= 64 * U * 1.5
