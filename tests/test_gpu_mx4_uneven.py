"""The attention over the 4-bit cache where a row's channels differ in size: encoder features have channels of large activation, and the
queries and gradients that meet them are small exactly there.

What is asked is the accuracy of a dot product in fp32, relative to the sizes of its own products and not to the operand's largest
value (u = 2^-24):
  scores and dP . x   |err| <= r * sum_c |a_c x_c|,  r = u (16 + 4 sqrt(D)): a few roundings a product, and D additions whose roundings
                      add up like a random walk (each at most u of a partial sum, which is at most sum_c |a_c x_c|; four deviations)
  delta = dP . P      likewise, with |P| <= sum_n A |x|: at most r * sum_n A_n sum_c |dP_c x_nc|
  weights             a score that is off by e changes a weight by 2 e relative to itself, plus 16 u for exponential, sum and quotient
  P, dq               sums over the tokens of weights times |x|, with those errors and the rounding of the sum, r' = u (16 + 4 sqrt(N))."""
import numpy as np
import pytest
import torch

from oracle import mx4_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _uneven(kind, D, rng):
    """Size of each channel of the tokens; queries and gradients are sized inversely."""
    size = np.ones(D)
    if kind == "lognormal":
        return np.exp(1.5 * rng.standard_normal(D))
    for lo in range(0, D, 32):                       # one channel of large activation in every group of 32
        size[lo + rng.integers(min(32, D - lo))] = kind
    return size


def _rows(shape, size, rng):
    return torch.from_numpy((rng.standard_normal(shape) / size).astype(np.float32))


FORMS = [(3, 70, 100, 3), (2, 197, 768, 8), (2, 197, 768, 16), (3, 100, 1152, 12), (2, 130, 384, 33), (2, 65, 2048, 8), (1, 70, 4096, 4), (1, 3000, 256, 8)]


@pytest.mark.parametrize("B,N,D,Q", FORMS)
@pytest.mark.parametrize("kind", [1e2, 1e3, 1e4, "lognormal"])
@pytest.mark.parametrize("per_image", [False, True])
def test_rows_of_uneven_channels(B, N, D, Q, kind, per_image):
    from efficient_probing_amd import mx4
    rng = np.random.default_rng(B + N + D + Q)
    size = _uneven(kind, D, rng)
    codes, scales = O.quantize(rng.standard_normal((B, N, D)) * size)
    x = O.dequantize(codes, scales, D)
    c = mx4.Mx4Tokens(torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV), D)
    q = _rows((B, Q, D) if per_image else (Q, D), size, rng)
    dP = _rows((B, Q, D), size, rng)
    scale = D ** -0.5
    qb, g = np.broadcast_to(q.double().numpy(), (B, Q, D)), dP.double().numpy()
    ln = np.full(B, N)
    Pr, Sr, Ar, dqr, _ = O.attention(x, ln, qb, scale, g)
    P, S, ML = mx4.pool_forward(c, q.to(DEV), scale, per_image_queries=per_image)
    r, rn = U * (16 + 4 * D ** 0.5), U * (16 + 4 * N ** 0.5)
    ax = np.abs(x).transpose(0, 2, 1)
    eS = r * scale * (np.abs(qb) @ ax)
    over = lambda got, want, lim: float((np.abs(got.double().cpu().numpy() - want) / (lim + 1e-30)).max())
    assert over(S, Sr, eS) <= 1.0, over(S, Sr, eS)
    relA = 2 * eS.max(-1, keepdims=True) + 16 * U
    lim = (relA + rn) * (Ar @ np.abs(x))
    assert over(P, Pr, lim) <= 1.0, over(P, Pr, lim)
    dq = mx4.pool_backward(c, S, ML, dP.to(DEV), scale, P=P, per_image_queries=per_image)
    mag = np.abs(g) @ ax                                                  # sizes of the products of dP . x
    magd = (Ar * mag).sum(-1, keepdims=True)
    dA = g @ x.transpose(0, 2, 1)
    dS = np.abs(dA - (Ar * dA).sum(-1, keepdims=True))
    eW = Ar * (relA * (dS + magd) + (r + rn) * (mag + magd))              # (delta carries P's error: relA + rn of its products)
    lim = scale * (eW @ np.abs(x) + rn * ((Ar * dS) @ np.abs(x)))
    want = dqr
    if not per_image:
        lim, want = lim.sum(0), want.sum(0)
    assert over(dq, want, lim) <= 1.0, over(dq, want, lim)


@pytest.mark.parametrize("B,N,D,Q", [(2, 70, 256, 8), (2, 70, 200, 16), (2, 70, 2048, 5)])
def test_powers_of_two_pass_through(B, N, D, Q):
    """Gradients and queries times a power of two: the same bits, moved (terms, weights and sums all scale)."""
    from efficient_probing_amd import mx4
    g = torch.Generator().manual_seed(D)
    c = mx4.quantize_tokens(torch.randn(B, N, D, generator=g).to(DEV))
    q, dP = torch.randn(Q, D, generator=g).to(DEV), torch.randn(B, Q, D, generator=g).to(DEV)
    P, S, ML = mx4.pool_forward(c, q, 0.125)
    dq = mx4.pool_backward(c, S, ML, dP, 0.125, P=P)
    for k in (-60, -20, 20, 60):
        assert torch.equal(mx4.pool_backward(c, S, ML, dP * 2.0 ** k, 0.125, P=P), dq * 2.0 ** k)
        for a, b in zip(mx4.pool_forward(c, q * 2.0 ** k, 0.125 * 2.0 ** -k), (P, S, ML)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("D", [256, 2048])
def test_rows_at_the_ends_of_fp32(D):
    """Rows near fp32's largest and smallest values stay finite and right; a row with an infinity or a NaN spoils its own query alone."""
    from efficient_probing_amd import mx4
    x = torch.zeros(1, 40, D)
    x[0, :, 5] = torch.arange(40) % 5 - 2.0
    c = mx4.quantize_tokens(x.to(DEV))
    q = torch.zeros(6, D)
    q[0, 5], q[1, 5], q[2, 5], q[3, 5], q[4, 7], q[5, 9] = 3.0e38, 2.0 ** -120, 1.5 * 2.0 ** -126, 1.0, float("inf"), float("nan")
    P, S, ML = mx4.pool_forward(c, q.to(DEV), 0.25)
    want = (q[:4, 5].double() * 0.25)[:, None] * x[0, :, 5].double()
    got = S[0, :4].double().cpu()
    # a term's scale is a normal number, 2^(5 t - 127) at least for the t-th last: the last term's grid is 2^(5 - 127) / 8 = 2^-125 (wide rows
    # alike), so that up to 2^-126 of a channel is lost whatever its size; times |x| <= 2
    assert ((got - want).abs() <= 2.0 ** -23 * want.abs() + 2.0 ** -126 * 2.0).all()
    assert bool(torch.isfinite(P[0, :4]).all()) and bool(torch.isnan(P[0, 4:]).all())
