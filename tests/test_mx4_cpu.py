"""The 4-bit token cache and the top-logit distillation without a GPU: what the calls refuse, and the oracles against hand-made
values and differences."""
import numpy as np
import pytest
import torch

from oracle import distill_oracle, mx4_oracle


def _cache(M=2, N=5, D=100, **kw):
    from efficient_probing_amd import mx4
    cb, sb = mx4.row_bytes(D)
    return mx4.Mx4Tokens(torch.zeros(M, N, cb, dtype=torch.uint8), torch.full((M, N, sb), 127, dtype=torch.uint8), D, **kw)


def test_cache_layout_and_views():
    from efficient_probing_amd import mx4
    assert mx4.row_bytes(768) == (384, 24) and mx4.row_bytes(100) == (64, 4) and mx4.row_bytes(129) == (128, 8)
    c = _cache(6, 5, 130, lengths=torch.tensor([0, 1, 2, 3, 4, 5], dtype=torch.int32))
    assert tuple(c.shape) == (6, 5, 130) and len(c) == 6 and c.nbytes == 6 * 5 * (128 + 8)
    b = c.select(torch.tensor([3, 3, 0], dtype=torch.int32))
    assert tuple(b.shape) == (3, 5, 130) and b.codes.data_ptr() == c.codes.data_ptr()
    v = c.tokens(1, 5)
    assert tuple(v.shape) == (6, 4, 130) and v.lengths.tolist() == [0, 0, 1, 2, 3, 4]
    assert v.codes.data_ptr() == c.codes.data_ptr() + 128 and c.lengths.tolist() == [0, 1, 2, 3, 4, 5]
    r = c.images(2, 4)
    assert tuple(r.shape) == (2, 5, 130) and r.lengths.tolist() == [2, 3]
    assert c.to("cpu") is c


@pytest.mark.parametrize("make", [
    lambda m: m.Mx4Tokens(torch.zeros(2, 5, 64, dtype=torch.int8), torch.zeros(2, 5, 4, dtype=torch.uint8), 100),
    lambda m: m.Mx4Tokens(torch.zeros(2, 5, 64, dtype=torch.uint8), torch.zeros(2, 5, 4, dtype=torch.uint8), 130),
    lambda m: m.Mx4Tokens(torch.zeros(2, 5, 64, dtype=torch.uint8), torch.zeros(2, 4, 4, dtype=torch.uint8), 100),
    lambda m: m.Mx4Tokens(torch.zeros(2, 5, 128, dtype=torch.uint8)[..., ::2], torch.zeros(2, 5, 4, dtype=torch.uint8), 100),
    lambda m: m.Mx4Tokens(torch.zeros(2, 10, 64, dtype=torch.uint8)[:, ::2], torch.zeros(2, 5, 4, dtype=torch.uint8), 100),
    lambda m: m.Mx4Tokens(torch.zeros(1, 5, 64, dtype=torch.uint8).expand(2, 5, 64), torch.zeros(2, 5, 4, dtype=torch.uint8), 100),
    lambda m: m.Mx4Tokens(torch.zeros(0, 5, 64, dtype=torch.uint8), torch.zeros(0, 5, 4, dtype=torch.uint8), 100),
    lambda m: _cache(lengths=torch.zeros(2, dtype=torch.int64)),
    lambda m: _cache(lengths=torch.zeros(3, dtype=torch.int32)),
    lambda m: _cache().select(torch.zeros(3, dtype=torch.int64)),
    lambda m: _cache().select(torch.zeros((3, 1), dtype=torch.int32)),
    lambda m: _cache().select(torch.zeros(3, dtype=torch.int32)).select(torch.zeros(3, dtype=torch.int32)),
    lambda m: _cache().images(1, 3),
    lambda m: _cache().images(1, 1),
    lambda m: _cache().tokens(2, 6),
    lambda m: m.Mx4Tokens(torch.zeros(2, 5, 64, dtype=torch.uint8), torch.zeros(2, 5, 4, dtype=torch.uint8, device="meta"), 100),
])
def test_cache_refuses(make):
    from efficient_probing_amd import mx4
    with pytest.raises(ValueError):
        make(mx4)


def test_no_cpu_path():
    from efficient_probing_amd import distill, mx4
    c = _cache()
    for call in (lambda: mx4.quantize_tokens(torch.zeros(2, 5, 100)), lambda: mx4.dequantize_tokens(c),
                 lambda: mx4.pool_forward(c, torch.zeros(3, 100), 1.0), lambda: mx4.attention_pool(c, torch.zeros(3, 100), 1.0),
                 lambda: distill.topk_distillation(torch.zeros(2, 5), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_c_entries_refuse_on_the_host():
    """The C ABI checks its arguments before it touches the device."""
    import ctypes as C
    from efficient_probing_amd import _native as N
    lib = N.load()
    codes, scales = torch.zeros(2 * 5 * 64, dtype=torch.uint8), torch.zeros(2 * 5 * 4, dtype=torch.uint8)
    buf = torch.zeros(4096)
    ok = dict(codes=codes.data_ptr() // 16 * 16, scales=scales.data_ptr() // 4 * 4, codes_bstride=320, scales_bstride=20, M=2, B=2, N=5, D=100)
    need = lib.ep_mx4_pool_workspace_bytes(2, 5, 100, 3)
    assert need > 0 and lib.ep_mx4_pool_workspace_bytes(0, 5, 100, 3) == 0

    def fwd(q=buf.data_ptr(), Q=3, ws=buf.data_ptr() // 16 * 16, nb=need, **over):
        t = N.EPMx4Tokens(**{**ok, **over})
        return lib.ep_mx4_pool_forward(C.byref(t), q, 0, Q, 1.0, buf.data_ptr(), 0, 0, buf.data_ptr() // 16 * 16, ws, nb, 0)

    assert fwd(codes=0) == -1 and fwd(q=0) == -1 and fwd(Q=0) == -1 and fwd(N=0) == -1
    assert fwd(B=3) == -1                                          # three images of a cache of two, without an index
    assert fwd(codes_bstride=304) == -2 and fwd(D=4097, codes_bstride=1 << 20, scales_bstride=1 << 20) == -2
    assert fwd(codes_bstride=328) == -3 and fwd(scales_bstride=22) == -3
    assert fwd(nb=need - 1) == -4 and "workspace" in N.last_error()
    t = N.EPMx4Tokens(**ok)
    assert lib.ep_mx4_dequantize(C.byref(t), buf.data_ptr() // 16 * 16, 7, 0) == -5
    assert lib.ep_mx4_quantize(buf.data_ptr(), 9, 500, 100, 2, 5, 100, ok["codes"], ok["scales"], 320, 20, 0) == -5
    bwd = lambda per, acc, sst=8: lib.ep_mx4_pool_backward(C.byref(t), 3, 1.0, buf.data_ptr() // 16 * 16, sst, buf.data_ptr() // 16 * 16, 0, buf.data_ptr(), buf.data_ptr(),
                                                    per, acc, buf.data_ptr() // 16 * 16, need, 0)
    assert bwd(1, 1) == -5 and bwd(0, 0, 6) == -3 and bwd(0, 0, 4) == -3
    d = dict(logits=buf.data_ptr(), dtype=0, ldl=10, B=2, C=10, K=3, R=2, teacher_values=buf.data_ptr(), ldv=3, teacher_index=buf.data_ptr(), ldi=3,
             temperature=1.0, alpha=1.0, grad_scale=1.0, loss_rows=buf.data_ptr())
    dist = lambda **over: lib.ep_distill_topk(C.byref(N.EPDistillArgs(**{**d, **over})), buf.data_ptr(), 1 << 20, 0)
    assert dist(logits=0) == -1 and dist(B=0) == -1 and dist(alpha=0.5) == -1 and dist(temperature=0.0) == -1 and dist(R=1) == -1
    assert dist(temperature=float("nan")) == -1 and dist(alpha=float("nan")) == -1
    assert dist(ldl=9) == -2 and dist(K=1025, ldv=2000, ldi=2000) == -2 and dist(C=(1 << 20) + 1, ldl=1 << 21) == -2 and dist(dtype=3) == -5


def test_oracle_values_by_hand():
    x = np.zeros((1, 1, 32))
    x[0, 0, :12] = [6, -6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, 0.24, 4.9]     # amax 6: exponent 0
    codes, scales = mx4_oracle.quantize(x)
    assert codes.shape == (1, 1, 64) and scales[0, 0].tolist() == [127, 2, 2, 2]
    got = mx4_oracle.dequantize(codes, scales, 32)[0, 0, :12]
    assert got.tolist() == [6, -6, 0, 1, 1, 2, 2, 4, 4, 0, 0, 4]                        # ties go to the even code
    x[0, 0, 0] = 7.0                                                                   # 1.75 * 4: one exponent up
    assert mx4_oracle.quantize(x)[1][0, 0, 0] == 128
    x[0, 0, 0] = 6.999
    assert mx4_oracle.quantize(x)[1][0, 0, 0] == 127
    x[0, 0, 0] = np.inf
    assert mx4_oracle.quantize(x)[1][0, 0, 0] == 255 and np.isnan(mx4_oracle.dequantize(*mx4_oracle.quantize(x), 32)).all()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T,alpha", [(1.0, 1.0), (2.5, 0.3)])
def test_distillation_oracle_against_differences(T, alpha, tail):
    rng = np.random.default_rng(3)
    B, C, K = 4, 9, 4
    z, v = rng.standard_normal((B, C)), rng.standard_normal((B, K)) * 2
    idx = np.stack([rng.permutation(C)[:K] for _ in range(B)])
    idx[1, 2] = idx[1, 0]                        # a class twice
    idx[2, 1] = -1
    idx[3] = -1                                  # nothing listed
    t = rng.standard_normal(B) if tail else None
    tg = np.array([2, 0, -1, 5])
    loss, grad = distill_oracle.distill(z, v, idx, tg, t, T, alpha)
    if not tail:
        assert alpha < 1 or loss[3] == 0
    h = 1e-6
    for b in range(B):
        for i in range(C):
            zp, zm = z.copy(), z.copy()
            zp[b, i] += h; zm[b, i] -= h
            d = (distill_oracle.distill(zp, v, idx, tg, t, T, alpha)[0][b] - distill_oracle.distill(zm, v, idx, tg, t, T, alpha)[0][b]) / (2 * h)
            assert abs(d - grad[b, i]) < 1e-8


def test_attention_oracle_against_differences():
    rng = np.random.default_rng(4)
    x, q, dP = rng.standard_normal((2, 5, 7)), rng.standard_normal((2, 3, 7)), rng.standard_normal((2, 3, 7))
    ln = np.array([5, 3])
    _, _, _, dq, _ = mx4_oracle.attention(x, ln, q, 0.4, dP)
    h = 1e-6
    for pos in np.ndindex(q.shape):
        qp, qm = q.copy(), q.copy()
        qp[pos] += h; qm[pos] -= h
        d = ((mx4_oracle.attention(x, ln, qp, 0.4)[0] - mx4_oracle.attention(x, ln, qm, 0.4)[0]) * dP).sum() / (2 * h)
        assert abs(d - dq[pos]) < 1e-8


@pytest.mark.parametrize("D", [100, 192, 1000, 1088, 2500, 4090])
def test_workspace_does_not_grow_with_the_batch(D):
    """Operand rows are read where they lie, also where a row is not whole 128-channel blocks: what is left is the workgroups' partial
    gradients (at most 16 waves on each of a chip's compute units, taken as 304 at most)."""
    from efficient_probing_amd import _native as N
    lib = N.load()
    for Q in (1, 8, 32):
        sizes = {lib.ep_mx4_pool_workspace_bytes(B, 20, D, Q) for B in (8192, 16384, 65536)}
        assert len(sizes) == 1 and 0 < sizes.pop() <= 304 * 8 * Q * D * 4 + 256
