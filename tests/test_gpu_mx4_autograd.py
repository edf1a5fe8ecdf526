"""The differentiable calls over a 4-bit cache when the cache changes between forward and backward: an error, as for any saved tensor."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _made(lengths=False):
    from efficient_probing_amd import mx4
    x = torch.randn(4, 20, 128, device=DEV)
    ln = torch.tensor([20, 3, 0, 7], dtype=torch.int32, device=DEV) if lengths else None
    return mx4.quantize_tokens(x, lengths=ln), torch.randn(3, 128, device=DEV, requires_grad=True)


def _write_again(mx4, c, idx):
    mx4.quantize_tokens(torch.randn(4, 20, 128, device=DEV), out=c)


def _write_a_range(mx4, c, idx):
    mx4.quantize_tokens(torch.randn(1, 20, 128, device=DEV), out=c.images(1, 2))


CHANGES = [_write_again, _write_a_range, lambda mx4, c, idx: c.codes.zero_(), lambda mx4, c, idx: c.scales.fill_(127), lambda mx4, c, idx: c.lengths.fill_(1),
           lambda mx4, c, idx: idx.fill_(0)]


@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("project", [False, True])
def test_a_cache_that_changed_is_an_error(change, project):
    from efficient_probing_amd import mx4
    c, q = _made(lengths=True)
    idx = torch.tensor([3, 0, 1], dtype=torch.int32, device=DEV)
    w = torch.randn(12, 128, device=DEV, requires_grad=True)
    out = mx4.pool_project(c.select(idx), q, w, 0.1) if project else mx4.attention_pool(c, q, 0.1, image_index=idx)
    change(mx4, c, idx)
    with pytest.raises(RuntimeError, match="modified"):
        out.sum().backward()


def test_reading_and_later_writes_are_no_change():
    from efficient_probing_amd import mx4
    c, q = _made()
    out = mx4.attention_pool(c, q, 0.1)
    mx4.dequantize_tokens(c)
    mx4.quantize_tokens(torch.randn(4, 20, 128, device=DEV))                # another cache
    out.sum().backward(retain_graph=True)
    first = q.grad.clone()
    out.sum().backward()
    assert torch.equal(q.grad, 2 * first)
    mx4.quantize_tokens(torch.randn(4, 20, 128, device=DEV), out=c)
    mx4.attention_pool(c, q, 0.1).sum().backward()


def test_a_cache_made_in_inference_mode():
    from efficient_probing_amd import mx4
    with torch.inference_mode():
        c, _ = _made(lengths=True)
        mx4.quantize_tokens(torch.randn(2, 20, 128, device=DEV), out=c.images(0, 2))
    mx4.quantize_tokens(torch.randn(1, 20, 128, device=DEV), out=c.images(2, 3))
    q = torch.randn(3, 128, device=DEV, requires_grad=True)
    mx4.attention_pool(c, q, 0.1).sum().backward()
    assert bool(torch.isfinite(q.grad).all())
