"""The 4-bit token cache and the attention over it against the float64 oracle.

Tolerances (u = 2^-24): quantising and reading back in bf16 / fp32 are exact.  A score is a sum of D products in fp32, off by about
u * sigma * sqrt(D) for scores of spread sigma (the partial sums are of size sigma, and their D roundings add up like a random walk);
a softmax weight is off by that relative to itself, plus a few u for the exponential and the sum, and so are the pooled rows:
|dP| <= u (16 + 4 (sigma + 1) sqrt(D)) * sum A |x|.  The gradient's weight A (dA - delta) carries the same relative errors on
terms of size A |dP| |x|, whose sum is the oracle's `mag`."""
import numpy as np
import pytest
import torch

from oracle import mx4_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _tokens(M, N, D, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(M, N, D, generator=g) * torch.exp(0.5 * torch.randn(D, generator=g)) + 0.2 * torch.randn(D, generator=g)).to(dtype)


def _cache(M, N, D, seed, lengths=None):
    from efficient_probing_amd import mx4
    codes, scales = O.quantize(_tokens(M, N, D, seed).numpy())
    c = mx4.Mx4Tokens(torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV), D,
                      lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV))
    return c, O.dequantize(codes, scales, D)


# ------------------------------------------------------------------------------------------------ writer and reader
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,N,D", [(1, 1, 1), (2, 3, 31), (1, 5, 32), (3, 7, 33), (2, 4, 100), (5, 17, 128), (2, 3, 130), (3, 16, 384), (2, 9, 1152), (1, 2, 4104)])
def test_quantize_is_exact(B, N, D, dtype):
    from efficient_probing_amd import mx4
    x = _tokens(B, N, D, B * 100 + D, dtype)
    c = mx4.quantize_tokens(x.to(DEV))
    codes, scales = O.quantize(x.double().numpy())
    assert np.array_equal(c.scales.cpu().numpy(), scales)
    assert np.array_equal(c.codes.cpu().numpy(), codes)
    want = O.dequantize(codes, scales, D)
    for out in (torch.bfloat16, torch.float32):
        assert np.array_equal(mx4.dequantize_tokens(c, out).double().cpu().numpy(), want)
    assert torch.equal(mx4.dequantize_tokens(c, torch.float16).cpu(), torch.from_numpy(want).to(torch.float16))


def test_quantize_hard_values():
    """Ties, the exponent's borders, the ends of the exponent range, subnormals, groups of zeros, infinities and NaN."""
    from efficient_probing_amd import mx4
    rows = []
    for e in (-149, -140, -126, -125, -124, -100, -1, 0, 1, 60, 124, 125, 126, 127):
        for top in (1.0, 1.25, 1.5, 1.7499999, 1.75, 1.9999999):
            v = np.array([0, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, .2499999, .2500001, .7499999, .7500001, 4.999999, 5.000001] + [0.0] * 18) * 2.0 ** -3
            v[-1] = top
            r = v * 2.0 ** e
            r[2::3] *= -1
            rows.append(np.float32(r))
    rows.append(np.zeros(32, np.float32))
    rows.append(np.float32([-0.0] * 32))
    for special in (np.inf, -np.inf, np.nan):
        r = np.linspace(-3, 3, 32).astype(np.float32)
        r[7] = special
        rows.append(r)
    x = np.stack(rows)
    x = np.concatenate([x, x[::-1]], 1)[None]                     # two groups a row: a bad one leaves its neighbour alone
    c = mx4.quantize_tokens(torch.from_numpy(x).to(DEV))
    codes, scales = O.quantize(x)
    assert np.array_equal(c.scales.cpu().numpy(), scales) and np.array_equal(c.codes.cpu().numpy(), codes)
    got = mx4.dequantize_tokens(c, torch.float32).double().cpu().numpy()
    assert np.array_equal(got, O.dequantize(codes, scales, 64), equal_nan=True)


def test_quantize_strides_and_ranges():
    from efficient_probing_amd import mx4
    big = torch.randn(4, 9, 200, device=DEV)
    views = [big[:, 1:], big[::2], big[:, ::2], big[..., :100], big[..., 3:103], big.transpose(0, 1), big[:1].expand(3, 9, 200), big.transpose(1, 2)]
    for v in views:
        a, b = mx4.quantize_tokens(v), mx4.quantize_tokens(v.contiguous())
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    cache = mx4.empty_cache(7, 9, 200, DEV)
    cache.codes.fill_(0xAB); cache.scales.fill_(77)
    mx4.quantize_tokens(big, out=cache.images(2, 6))
    want = mx4.quantize_tokens(big)
    assert torch.equal(cache.codes[2:6], want.codes) and torch.equal(cache.scales[2:6], want.scales)
    for lo, hi in ((0, 2), (6, 7)):                               # the rows beside the range stay as they were
        assert bool((cache.codes[lo:hi] == 0xAB).all()) and bool((cache.scales[lo:hi] == 77).all())
    idx = torch.tensor([5, 2, 2, -1, 7, 3], dtype=torch.int32, device=DEV)
    got = mx4.dequantize_tokens(cache, torch.float32, image_index=idx)
    ref = mx4.dequantize_tokens(want, torch.float32)
    for r, src in enumerate((3, 0, 0, None, None, 1)):
        assert bool(torch.isnan(got[r]).all()) if src is None else torch.equal(got[r], ref[src])
    tok = mx4.dequantize_tokens(cache.tokens(1, 9), torch.float32, image_index=idx[:3])
    assert torch.equal(tok, got[:3, 1:])


# ------------------------------------------------------------------------------------------------ attention
def _check(c, x, q, scale, per_image=False, index=None, lengths=None, seed=0, P_in=True):
    """Forward and backward of one call against the oracle; returns the outputs."""
    from efficient_probing_amd import mx4
    B, N, D = (len(index) if index is not None else x.shape[0]), x.shape[1], x.shape[2]
    Q = q.shape[-2]
    src = np.arange(B) if index is None else np.asarray(index)
    ln = np.full(B, N) if lengths is None else np.clip(np.asarray(lengths), 0, N)[src]
    idx = None if index is None else torch.tensor(index, dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(seed + 17)
    dP = torch.randn(B, Q, D, generator=g)
    qb = q.double().numpy() if per_image else np.broadcast_to(q.double().numpy(), (B, Q, D))
    xs = x[src]
    Pr, Sr, Ar, dqr, mag = O.attention(xs, ln, qb, scale, dP.double().numpy())
    qg = q.to(DEV)
    P, S, ML = mx4.pool_forward(c, qg, scale, per_image_queries=per_image, image_index=idx)
    P2, none, ML2 = mx4.pool_forward(c, qg, scale, per_image_queries=per_image, image_index=idx, need_scores=False)
    assert none is None and torch.equal(P, P2) and torch.equal(ML, ML2)
    fin = np.isfinite(Sr)
    sigma = float(np.abs(Sr[fin]).max()) if fin.any() else 0.0
    rel = U * (16 + 4 * (sigma + 1) * D ** 0.5)
    Sg, Pg = S.double().cpu().numpy(), P.double().cpu().numpy()
    assert np.array_equal(np.isneginf(Sg), ~fin)
    assert np.abs(Sg[fin] - Sr[fin]).max(initial=0.0) <= rel
    size = np.einsum("bqn,bnd->bqd", Ar, np.abs(np.where(np.arange(N)[None, :, None] < ln[:, None, None], xs, 0.0)))
    assert (np.abs(Pg - Pr) <= rel * size + 1e-30).all(), float((np.abs(Pg - Pr) / (rel * size + 1e-30)).max())
    m, l = ML[..., 0].double().cpu().numpy(), ML[..., 1].double().cpu().numpy()
    for b in range(B):
        if ln[b] == 0:
            assert (m[b] == 0).all() and (l[b] == 0).all() and (Pg[b] == 0).all()
        else:
            assert np.array_equal(m[b], Sg[b].max(-1))
            assert (np.abs(l[b] - np.exp(Sr[b] - Sr[b].max(-1, keepdims=True)).sum(-1)) <= 2 * rel * l[b]).all()
    if not P_in:
        ML[..., 2] = (dP.double() * torch.from_numpy(Pr)).sum(-1).float().to(DEV)
    dq = mx4.pool_backward(c, S, ML, dP.to(DEV), scale, P=P if P_in else None, per_image_queries=per_image, image_index=idx)
    want, bound = (dqr, mag) if per_image else (dqr.sum(0), mag.sum(0))
    got = dq.double().cpu().numpy()
    assert (np.abs(got - want) <= rel * bound + 1e-30).all(), float((np.abs(got - want) / (rel * bound + 1e-30)).max())
    return P, S, ML, dq


SHAPES = [(1, 1, 1, 1), (2, 1, 5, 3), (3, 2, 32, 1), (2, 15, 100, 5), (2, 16, 128, 8), (3, 17, 128, 9), (2, 31, 130, 16), (2, 33, 256, 17), (4, 63, 384, 8),
          (2, 65, 384, 32), (3, 197, 384, 8), (2, 197, 640, 33), (3, 256, 768, 8), (2, 129, 768, 48), (2, 257, 1024, 16), (2, 100, 1152, 12), (1, 300, 1408, 4),
          (2, 70, 2048, 8), (2, 50, 4096, 4), (1, 35, 4090, 33), (1, 2500, 128, 8), (1, 1031, 1024, 2), (40, 5, 64, 2)]


@pytest.mark.parametrize("B,N,D,Q", SHAPES)
@pytest.mark.parametrize("per_image", [False, True])
def test_attention(B, N, D, Q, per_image):
    c, x = _cache(B, N, D, D + N)
    g = torch.Generator().manual_seed(Q)
    q = torch.randn(*((B, Q, D) if per_image else (Q, D)), generator=g) * 1.5
    _check(c, x, q, D ** -0.5, per_image, seed=N)


@pytest.mark.parametrize("D", [1536, 1664, 1665, 1792, 1793, 1920, 1921, 2049, 2560, 2700, 3584, 3970, 4096])
@pytest.mark.parametrize("Q", [3, 13])
def test_every_cut_of_wide_rows(D, Q):
    """Rows around the border between the two forms of the kernel and around their slices, images of different lengths."""
    lengths = [0, 97, 1, 64, 33]
    c, x = _cache(5, 97, D, D, lengths)
    q = torch.randn(Q, D, generator=torch.Generator().manual_seed(Q)) * 1.5
    _check(c, x, q, D ** -0.5, False, [1, 4, 0, 3, 2, 1], lengths)


def test_more_images_than_compute_units_of_wide_rows():
    c, x = _cache(20, 40, 2100, 7)
    q = torch.randn(5, 2100, generator=torch.Generator().manual_seed(2))
    _check(c, x, q, 2100 ** -0.5, False, [i % 20 for i in range(600)])


@pytest.mark.parametrize("B,N,D,Q", [(6, 1, 64, 2), (7, 40, 130, 8), (6, 197, 384, 12), (5, 257, 1152, 8), (4, 90, 768, 32), (3, 40, 4096, 2)])
@pytest.mark.parametrize("per_image", [False, True])
def test_ragged_and_indexed(B, N, D, Q, per_image):
    """Lengths from none to all (and beyond, and negative: clamped), images picked through an index, one of them twice."""
    M = B + 3
    rng = np.random.default_rng(B + N)
    lengths = [0, N, N + 5, -2] + [int(v) for v in rng.integers(0, N + 1, M - 4)]
    c, x = _cache(M, N, D, D, lengths)
    index = [int(v) for v in rng.permutation(M)[:B]]
    index[0], index[1] = 0, 2
    index[-1] = index[1]
    g = torch.Generator().manual_seed(1)
    q = torch.randn(*((B, Q, D) if per_image else (Q, D)), generator=g) * 1.5
    _check(c, x, q, D ** -0.5, per_image, index, lengths)
    _check(c, x, q, D ** -0.5, per_image, index, lengths, P_in=False)


@pytest.mark.parametrize("amp", [1e-3, 30.0, 300.0])
def test_sharp_and_flat_scores(amp):
    """From near uniform weights to a softmax that a single token takes; the row maximum moves late in the image."""
    c, x = _cache(3, 200, 256, 5)
    q = torch.randn(8, 256, generator=torch.Generator().manual_seed(2)) * amp
    _check(c, x, q, 1 / 16)


def test_masked_rows_may_hold_anything():
    """NaN groups, infinite scales and stale codes behind an image's length leave everything else untouched."""
    from efficient_probing_amd import mx4
    lengths = [37, 0, 64, 5]
    c, x = _cache(4, 64, 200, 9, lengths)
    q = torch.randn(9, 200, generator=torch.Generator().manual_seed(2), ) * 1.5
    ref = _check(c, x, q, 200 ** -0.5, lengths=lengths)
    for m, n in enumerate(lengths):
        c.codes[m, n:] = 0x77
        c.scales[m, n:] = 255
        if n + 1 < 64:
            c.scales[m, n + 1] = 254
    got = _check(c, x, q, 200 ** -0.5, lengths=lengths)
    for a, b in zip(ref, got):
        assert torch.equal(a.nan_to_num(1.0), b.nan_to_num(1.0)) and not torch.isnan(b).any()
    c.scales[2, 3, 1] = 255                                       # a NaN among the tokens that count is seen, in its image alone
    P, _, _ = mx4.pool_forward(c, q.to(DEV), 200 ** -0.5)
    assert bool(torch.isnan(P[2]).all()) and torch.equal(P[[0, 1, 3]], ref[0][[0, 1, 3]])


def test_index_outside_the_cache():
    from efficient_probing_amd import mx4
    c, x = _cache(3, 20, 96, 9)
    q = torch.randn(4, 96, device=DEV)
    idx = torch.tensor([1, -1, 3, 2, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV)
    P, S, ML = mx4.pool_forward(c, q, 0.1, image_index=idx)
    bad = [1, 2, 4, 5]
    assert bool(torch.isnan(P[bad]).all()) and not torch.isnan(P[[0, 3]]).any()
    good = torch.tensor([1, 2], dtype=torch.int32, device=DEV)
    Pg, Sg, MLg = mx4.pool_forward(c, q, 0.1, image_index=good)
    assert torch.equal(P[[0, 3]], Pg)
    dP = torch.randn(6, 4, 96, device=DEV)
    dq = mx4.pool_backward(c, S, ML, dP, 0.1, P=P, image_index=idx)
    dg = mx4.pool_backward(c, Sg, MLg, dP[[0, 3]].contiguous(), 0.1, P=Pg, image_index=good)
    torch.testing.assert_close(dq, dg, rtol=1e-5, atol=1e-5)
    per = mx4.pool_backward(c, S, ML, dP, 0.1, P=P, image_index=idx, per_image_queries=True)
    assert bool((per[bad] == 0).all())


def test_views_accumulate_and_repeat():
    from efficient_probing_amd import mx4
    N, D, Q = 50, 300, 6
    c, x = _cache(5, N, D, 3, [50, 0, 1, 2, 33])
    q = torch.randn(Q, D, generator=torch.Generator().manual_seed(2)) * 1.5
    v = c.tokens(1, N)                                            # without [CLS]
    P, S, ML, dq = _check(v, x[:, 1:], q, D ** -0.5, lengths=[49, 0, 0, 1, 32])
    _check(c.images(1, 4), x[1:4], q, D ** -0.5, lengths=[0, 1, 2])
    dP = torch.randn(5, Q, D, device=DEV)
    a = mx4.pool_backward(v, S, ML, dP, 0.3, P=P)
    start = torch.randn(Q, D, device=DEV)
    b = start.clone()
    assert mx4.pool_backward(v, S, ML, dP, 0.3, P=P, dq=b, accumulate=True) is b
    torch.testing.assert_close(b, a + start, rtol=1e-6, atol=1e-6)
    for _ in range(3):                                            # the same bits every time
        assert torch.equal(a, mx4.pool_backward(v, S, ML, dP, 0.3, P=P))
        assert torch.equal(P, mx4.pool_forward(v, q.to(DEV), D ** -0.5)[0])


def test_offsets_beyond_32_bits():
    """Images behind the first 4 GiB of a cache."""
    from efficient_probing_amd import mx4
    N, D = 197, 1024
    M = (1 << 32) // (N * 512) + 8
    c = mx4.empty_cache(M, N, D, DEV)
    small, x = _cache(3, N, D, 4)
    c.codes[M - 3:] = small.codes
    c.scales[M - 3:] = small.scales
    idx = torch.tensor([M - 1, M - 3], dtype=torch.int32, device=DEV)
    q = torch.randn(8, D, device=DEV)
    P, S, ML = mx4.pool_forward(c, q, D ** -0.5, image_index=idx)
    Ps, Ss, MLs = mx4.pool_forward(small, q, D ** -0.5, image_index=torch.tensor([2, 0], dtype=torch.int32, device=DEV))
    assert torch.equal(P, Ps) and torch.equal(S, Ss)
    back = mx4.dequantize_tokens(c, torch.float32, image_index=idx)
    assert np.array_equal(back.double().cpu().numpy(), x[[2, 0]])
    dP = torch.randn(2, 8, D, device=DEV)
    a = mx4.pool_backward(c, S, ML, dP, 1.0, P=P, image_index=idx)
    b = mx4.pool_backward(small, Ss, MLs, dP, 1.0, P=Ps, image_index=torch.tensor([2, 0], dtype=torch.int32, device=DEV))
    assert torch.equal(a, b)


def test_long_axis_few_images():
    """A token axis that is split over many workgroups and joined again."""
    for B, N, D, Q, per in ((1, 70001, 64, 3, False), (2, 20011, 384, 16, True), (1, 9000, 1024, 1, False)):
        c, x = _cache(B, N, D, N, None)
        q = torch.randn(*((B, Q, D) if per else (Q, D)), generator=torch.Generator().manual_seed(2)) * 1.5
        _check(c, x, q, D ** -0.5, per)
    c, x = _cache(2, 12000, 128, 7, [11999, 40])
    _check(c, x, torch.randn(5, 128, generator=torch.Generator().manual_seed(2)), 0.1, lengths=[11999, 40])


def test_autograd_streams_and_graphs():
    from efficient_probing_amd import mx4
    c, x = _cache(6, 77, 384, 11)
    q0 = torch.randn(8, 384, device=DEV)
    w = torch.randn(6, 8, 384, device=DEV)

    def eager():
        q = q0.clone().requires_grad_(True)
        P = mx4.attention_pool(c, q, 0.05)
        (P * w).sum().backward()
        return P.detach(), q.grad
    P, gq = eager()
    Pf, S, ML = mx4.pool_forward(c, q0, 0.05)
    assert torch.equal(P, Pf) and torch.equal(gq, mx4.pool_backward(c, S, ML, w, 0.05, P=Pf))
    q16 = q0.to(torch.bfloat16).requires_grad_(True)
    mx4.attention_pool(c, q16, 0.05).sum().backward()
    assert q16.grad.dtype == torch.bfloat16
    per = q0.expand(6, 8, 384).clone().requires_grad_(True)
    (mx4.attention_pool(c, per, 0.05, per_image_queries=True) * w).sum().backward()
    torch.testing.assert_close(per.grad.sum(0), gq, rtol=1e-4, atol=1e-5 * float(gq.abs().max()))
    with torch.no_grad():
        assert torch.equal(mx4.attention_pool(c, q0, 0.05), P)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        P2, g2 = eager()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(P, P2) and torch.equal(gq, g2)
    # captured: forward and backward, two graphs over the same buffers, replayed between eager work
    qs, dP = q0.clone(), w.clone()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            Pg, Sg, MLg = mx4.pool_forward(c, qs, 0.05)
            dg = mx4.pool_backward(c, Sg, MLg, dP, 0.05, P=Pg)
        graphs.append((gr, Pg, dg))
    for k in range(4):
        qs.copy_(q0 * (1 + k))
        Pe, Se, MLe = mx4.pool_forward(c, qs, 0.05)
        de = mx4.pool_backward(c, Se, MLe, dP, 0.05, P=Pe)
        for gr, Pg, dg in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for gr, Pg, dg in graphs:
            assert torch.equal(Pg, Pe) and torch.equal(dg, de)


@pytest.mark.parametrize("call", [
    lambda m, c: m.pool_forward(c, torch.zeros(3, 99, device=DEV), 1.0),
    lambda m, c: m.pool_forward(c, torch.zeros(2, 3, 100, device=DEV), 1.0),
    lambda m, c: m.pool_forward(c, torch.zeros(4, 3, 100, device=DEV), 1.0, per_image_queries=True),
    lambda m, c: m.pool_forward(c, torch.zeros(0, 100, device=DEV), 1.0),
    lambda m, c: m.pool_forward(c, torch.zeros(3, 100, device=DEV), 1.0, image_index=torch.zeros(3, dtype=torch.int32)),
    lambda m, c: m.pool_forward(c, torch.zeros(3, 100, device=DEV), 1.0, image_index=torch.zeros(3, dtype=torch.int64, device=DEV)),
    lambda m, c: m.dequantize_tokens(c, torch.float64),
    lambda m, c: m.quantize_tokens(torch.zeros(2, 5, 100, device=DEV), out=c),
    lambda m, c: m.quantize_tokens(torch.zeros(3, 5, 100, device=DEV), out=c.select(torch.zeros(3, dtype=torch.int32, device=DEV))),
    lambda m, c: m.quantize_tokens(torch.zeros(5, 100, device=DEV)),
    lambda m, c: m.pool_backward(c, torch.zeros(3, 2, 5, device=DEV), torch.zeros(3, 2, 4, device=DEV), torch.zeros(3, 2, 99, device=DEV), 1.0),
    lambda m, c: m.pool_backward(c, torch.zeros(3, 2, 4, device=DEV), torch.zeros(3, 2, 4, device=DEV), torch.zeros(3, 2, 100, device=DEV), 1.0),
    lambda m, c: m.pool_backward(c, torch.zeros(3, 2, 5, device=DEV), torch.zeros(3, 2, 4, device=DEV), torch.zeros(3, 2, 100, device=DEV), 1.0, accumulate=True),
])
def test_refusals(call):
    from efficient_probing_amd import mx4
    c = mx4.quantize_tokens(torch.randn(3, 5, 100, device=DEV))
    with pytest.raises(ValueError):
        call(mx4, c)


def test_wide_rows_are_refused_by_the_attention():
    from efficient_probing_amd import mx4
    c = mx4.quantize_tokens(torch.randn(1, 2, 4104, device=DEV))
    with pytest.raises(ValueError, match="4096"):
        mx4.pool_forward(c, torch.zeros(1, 4104, device=DEV), 1.0)


def test_calls_larger_than_a_launch():
    """More than 2^30 pieces of eight channels in one call (images of one broadcast tensor; a cache read through an index)."""
    from efficient_probing_amd import mx4
    B, N, D = 530000, 4, 4096
    x = _tokens(1, N, D, 3)
    codes, scales = (torch.from_numpy(a).to(DEV) for a in O.quantize(x.numpy()))
    c = mx4.quantize_tokens(x.to(torch.float32).to(DEV).expand(B, N, D))
    for lo in (0, 2 ** 30 // (N * 512) - 1, B - 2):
        assert bool((c.codes[lo:lo + 2] == codes).all()) and bool((c.scales[lo:lo + 2] == scales).all())
    del c
    back = mx4.dequantize_tokens(mx4.Mx4Tokens(codes, scales, D), torch.bfloat16, torch.zeros(B, dtype=torch.int32, device=DEV))
    want = mx4.dequantize_tokens(mx4.Mx4Tokens(codes, scales, D), torch.bfloat16)
    for lo in (0, 2 ** 30 // (N * 512) - 1, B - 2):
        assert bool((back[lo:lo + 2] == want).all())


@pytest.mark.parametrize("D,Q", [(1152, 12), (2048, 5)])
def test_captured_with_large_shared_memory(D, Q):
    from efficient_probing_amd import mx4
    c, x = _cache(3, 70, D, D)
    q, dP = torch.randn(Q, D, device=DEV), torch.randn(3, Q, D, device=DEV)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        P, S, ML = mx4.pool_forward(c, q, 0.05)
        dq = mx4.pool_backward(c, S, ML, dP, 0.05, P=P)
    for _ in range(3):
        q.normal_()
        Pe, Se, MLe = mx4.pool_forward(c, q, 0.05)
        de = mx4.pool_backward(c, Se, MLe, dP, 0.05, P=Pe)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(P, Pe) and torch.equal(S, Se) and torch.equal(dq, de)
