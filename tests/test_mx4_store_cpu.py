"""What needs no GPU of the compact store: teacher rows beside tokens of any type, the layout of a 4-bit store on disk, the criterion's
checks, and which head reads what."""
from argparse import Namespace

import numpy as np
import pytest
import torch

from efficient_probing_amd import distill, mx4, token_store as TS
from oracle import mx4_oracle


def test_teacher_topk_by_hand():
    z = torch.randn(5, 9, dtype=torch.float64, generator=torch.Generator().manual_seed(0)).float()
    v, i, t = distill.teacher_topk(z, 3, 2.0)
    assert v.dtype == torch.float32 and i.dtype == torch.int32 and torch.equal(z.gather(1, i.long()), v)
    rest = [[z[b, c].item() for c in range(9) if c not in i[b].tolist()] for b in range(5)]
    want = [np.log(np.exp(np.array(r, np.float64) / 2.0).sum()) for r in rest]
    assert np.allclose(t.numpy(), want, rtol=0, atol=2.0 ** -21)                 # six exponentials of size about 1, fp32
    assert all(v[b].min().item() >= max(rest[b]) for b in range(5))
    assert torch.isneginf(distill.teacher_topk(z, 9)[2]).all()
    for k, T in ((0, 1.0), (10, 1.0), (3, 0.0), (3, float("inf"))):
        with pytest.raises(ValueError):
            distill.teacher_topk(z, k, T)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_teacher_rows_follow_their_images(tmp_path, dtype, tail):
    rng = np.random.default_rng(0)
    n = 23
    tok, lab = rng.standard_normal((n, 4, 16), dtype=np.float32), rng.integers(0, 9, n)
    val, idx, tl = rng.standard_normal((n, 3), dtype=np.float32), rng.integers(0, 9, (n, 3)), rng.standard_normal(n).astype(np.float32)
    w = TS.TokenStoreWriter(str(tmp_path), 4, 16, shard_images=10, dtype=dtype, teacher_temperature=3.0)
    for lo, hi in ((0, 7), (7, 7), (7, 20), (20, n)):
        w.add(torch.from_numpy(tok[lo:hi]) if lo else tok[lo:hi], lab[lo:hi], teacher=(val[lo:hi], idx[lo:hi]) + ((tl[lo:hi],) if tail else ()))
    meta = w.close()
    assert meta["teacher"] == {"k": 3, "tail": tail, "temperature": 3.0} and "lengths" not in meta and [s["images"] for s in meta["shards"]] == [10, 10, 3]
    st = TS.ResidentTokenStore(str(tmp_path), "cpu")
    assert torch.equal(st.teacher.values, torch.from_numpy(val)) and torch.equal(st.teacher.index, torch.from_numpy(idx.astype(np.int32)))
    assert (st.teacher.tail is not None) == tail and (not tail or torch.equal(st.teacher.tail, torch.from_numpy(tl)))
    assert torch.equal(st.labels, torch.from_numpy(lab)) and torch.equal(st.tokens.float(), torch.from_numpy(tok).to(st.tokens.dtype).float())
    for rank in range(2):                                                      # each rank's rows are its own images'
        part = TS.ResidentTokenStore(str(tmp_path), "cpu", world=2, rank=rank)
        pick = np.r_[0:10, 20:23] if rank == 0 else np.r_[10:20]
        assert torch.equal(part.teacher.values, torch.from_numpy(val[pick])) and torch.equal(part.labels, torch.from_numpy(lab[pick]))
    crit = distill.TopKDistillation.from_store(st)
    assert crit.temperature == 3.0 and crit.alpha == 1.0 and not crit.state_dict()
    if tail:
        with pytest.raises(ValueError, match="temperature"):
            distill.TopKDistillation.from_store(st, temperature=1.0)
    else:
        assert distill.TopKDistillation.from_store(st, temperature=1.0).temperature == 1.0


def test_writer_refusals(tmp_path):
    tok, lab = np.zeros((4, 2, 8), np.float32), np.zeros(4, np.int64)
    w = TS.TokenStoreWriter(str(tmp_path), 2, 8)
    for bad in ((np.zeros((4, 3)),), (np.zeros((4, 3)), np.zeros((4, 2))), (np.zeros((3, 3)), np.zeros((3, 3))), (np.zeros(4), np.zeros(4)),
                (np.zeros((4, 3)), np.zeros((4, 3)), np.zeros(3)), (np.zeros((4, 3)), np.full((4, 3), 2 ** 32 + 1))):
        with pytest.raises(ValueError):
            w.add(tok, lab, teacher=bad)
    with pytest.raises(ValueError, match="mxfp4"):
        w.add(tok, lab, lengths=np.ones(4))
    w.add(tok, lab, teacher=(np.zeros((4, 3)), np.zeros((4, 3))))
    for bad in (None, (np.zeros((4, 2)), np.zeros((4, 2))), (np.zeros((4, 3)), np.zeros((4, 3)), np.zeros(4))):
        with pytest.raises(ValueError):
            w.add(tok, lab, teacher=bad)
    assert w.close()["total_images"] == 4
    with pytest.raises(NotImplementedError):
        TS.TokenStoreWriter(str(tmp_path), 2, 8, dtype="int4")
    with pytest.raises(ValueError, match="no teacher"):
        distill.TopKDistillation.from_store(TS.ResidentTokenStore.from_tensors(torch.zeros(2, 3, 8), torch.zeros(2)))


@pytest.mark.parametrize("lengths", [False, True])
def test_four_bit_store_on_disk(tmp_path, lengths, monkeypatch):
    """The files of an mxfp4 store, written with the oracle's codes in place of the GPU's."""
    N, D, n = 3, 40, 11
    rng = np.random.default_rng(1)
    tok, lab, ln = rng.standard_normal((n, N, D), dtype=np.float32), rng.integers(0, 5, n), rng.integers(0, N + 1, n)
    codes, scales = (torch.from_numpy(a) for a in mx4_oracle.quantize(tok))
    monkeypatch.setattr(torch.Tensor, "to", lambda self, *a, _to=torch.Tensor.to, **k: self if a[:1] == ("cuda",) else _to(self, *a, **k))
    monkeypatch.setattr(mx4, "quantize_tokens", lambda x: mx4.Mx4Tokens(*(torch.from_numpy(a) for a in mx4_oracle.quantize(x.numpy())), D))
    w = TS.TokenStoreWriter(str(tmp_path), N, D, shard_images=4, dtype="mxfp4")
    for lo in (0, 5, 10):
        w.add(tok[lo:lo + 5], lab[lo:lo + 5], lengths=ln[lo:lo + 5] if lengths else None)
    with pytest.raises(ValueError):
        w.add(tok[:1], lab[:1], lengths=None if lengths else ln[:1])
    if lengths:
        with pytest.raises(ValueError):
            w.add(tok[:1], lab[:1], lengths=[N + 1])
    meta = w.close()
    assert meta["dtype"] == "mxfp4" and bool(meta.get("lengths")) == lengths
    assert (tmp_path / "tokens-00000.bin").stat().st_size == 4 * N * 64 and (tmp_path / "scales-00000.bin").stat().st_size == 4 * N * 4
    st = TS.ResidentTokenStore(str(tmp_path), "cpu", seed=2)
    assert st.dtype == "mxfp4" and tuple(st.tokens.shape) == (n, N, D) and torch.equal(st.tokens.codes, codes) and torch.equal(st.tokens.scales, scales)
    assert (st.tokens.lengths is None) != lengths and (not lengths or torch.equal(st.tokens.lengths, torch.from_numpy(ln.astype(np.int32))))
    for cache, idx, tgt in st.batches(4):
        assert cache is st.tokens and tuple(cache.select(idx).shape) == (4, N, D) and torch.equal(tgt, st.labels[idx.long()])
    with pytest.raises(ValueError, match="open_shard_arrays"):
        TS.open_shard(str(tmp_path), meta, meta["shards"][0])
    with pytest.raises(ValueError, match="tables"):
        st.table("token_stats", 1e-6)
    with pytest.raises(ValueError, match="cache, not a batch"):
        TS.ResidentTokenStore.from_tensors(st.tokens.select(torch.zeros(2, dtype=torch.int32)), torch.zeros(2))
    empty = TS.ResidentTokenStore(str(tmp_path), "cpu", world=8, rank=7)
    assert empty.num_images == 0 and not empty.tokens.codes.any() and list(empty.batches(4)) == []


def test_criterion_refusals():
    v, i = torch.zeros(6, 3), torch.zeros(6, 3, dtype=torch.int64)
    for kw in (dict(temperature=0.0), dict(temperature=float("inf")), dict(alpha=1.5), dict(teacher_tail=torch.zeros(5))):
        with pytest.raises(ValueError):
            distill.TopKDistillation(v, i, **kw)
    with pytest.raises(ValueError):
        distill.TopKDistillation(v, i[:, :2])
    c = distill.TopKDistillation(v, i)
    with pytest.raises(ValueError, match="image_index"):
        c._rows(4, None)
    assert c._rows(6, None) is None and c._rows(2, torch.tensor([5, 5])).dtype == torch.int32
    assert c._rows(2, torch.tensor([2 ** 32 + 5, -2 ** 40])).tolist() == [2 ** 31 - 1, -1]          # out of range, not wrapped into it
    i[0, 0] = 2 ** 32 + 1
    assert distill.TopKDistillation(v, i).teacher_index[0, 0] == distill.MAX_CLASSES
    with pytest.raises(ValueError, match="integers"):
        distill.TopKDistillation(v, v)


def test_tables_are_not_looked_up_in_a_store_of_codes():
    """An engine that has seen a 4-bit store is then called with a batch of its own."""
    from efficient_probing_amd.engine import CaeHeadEngine
    cache = mx4.Mx4Tokens(torch.zeros(3, 2, 64, dtype=torch.uint8), torch.zeros(3, 2, 4, dtype=torch.uint8), 100)
    eng = CaeHeadEngine.__new__(CaeHeadEngine)
    eng._store = TS.ResidentTokenStore.from_tensors(cache, torch.zeros(3))
    assert eng._store_kinds
    eng._bind_store_tables(torch.zeros(3, 2, 100), torch.zeros(2, dtype=torch.int32))
    assert eng._bound_tables == {}


def test_who_reads_codes():
    from efficient_probing_amd import engine_finetune as EF, probe_heads
    made = {}
    for head in ("ep", "simpool", "all"):
        m = torch.nn.Module()
        m.head = torch.nn.Linear(64, 5)
        if head != "all":
            probe_heads.build_probe_head(m, Namespace(cls_features=head, ep_queries=4, d_out=1, nb_classes=5, num_heads=4))
        made[head] = EF._reads_parts(m)
    assert made == {"ep": True, "simpool": False, "all": False}
    cache = mx4.Mx4Tokens(torch.zeros(3, 2, 64, dtype=torch.uint8), torch.zeros(3, 2, 4, dtype=torch.uint8), 100, lengths=torch.tensor([2, 1, 0], dtype=torch.int32))
    idx = torch.tensor([1], dtype=torch.int32)
    assert EF._batch_tokens(cache, idx, True, None) == (cache, idx)
    with pytest.raises(ValueError, match="EP head"):
        EF._batch_tokens(cache, idx, False, None)
    x = torch.zeros(2, 3, 4)
    assert EF._batch_tokens(x, idx, False, None) == (x, idx)


def test_writer_takes_what_it_took(tmp_path):
    """Tokens as nested lists, as integers or doubles, and torch tensors of any floating type; teacher rows likewise."""
    tok = [[[1.0, 2.0, 3.0, 4.0, 5.0, 6.0, 7.0, 8.0]], [[0.5] * 8]]
    x = torch.tensor(tok)
    w = TS.TokenStoreWriter(str(tmp_path / "a"), 1, 8)
    for t in (tok, np.array(tok, np.float64), np.array(tok).astype(np.int32), x, x.double(), x.to(torch.bfloat16), x.half(), x.transpose(0, 1).contiguous().transpose(0, 1)):
        w.add(t, [3, 4])
    assert w.close()["total_images"] == 16
    st = TS.ResidentTokenStore(str(tmp_path / "a"), "cpu")
    for lo in range(0, 16, 2):
        assert torch.equal(st.tokens[lo:lo + 2], x if lo != 4 else x.floor())
    w = TS.TokenStoreWriter(str(tmp_path / "b"), 1, 8)
    w.add(x.to(torch.bfloat16), [0, 1], teacher=(torch.tensor([[2.0, 1.0], [0.5, 0.25]], dtype=torch.bfloat16), [[4, 2], [0, 1]], torch.zeros(2, dtype=torch.bfloat16)))
    w.close()
    t = TS.ResidentTokenStore(str(tmp_path / "b"), "cpu").teacher
    assert t.values.tolist() == [[2.0, 1.0], [0.5, 0.25]] and t.index.tolist() == [[4, 2], [0, 1]] and t.tail.tolist() == [0.0, 0.0]
    with pytest.raises(AssertionError):
        w.add([[1.0] * 8], [0])


@pytest.mark.parametrize("T", [1e-20, 1e-40, 1e20, 3e38])
def test_temperatures_whose_square_or_inverse_leaves_fp32(T):
    """They gave losses of 0 times infinity."""
    import ctypes as C
    from efficient_probing_amd import _native as N
    v, i = torch.zeros(6, 3), torch.zeros(6, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="temperature"):
        distill.TopKDistillation(v, i, temperature=T)
    with pytest.raises(ValueError, match="temperature"):
        distill.teacher_topk(torch.zeros(2, 5), 3, T)
    buf = torch.zeros(64)
    a = N.EPDistillArgs(logits=buf.data_ptr(), dtype=0, ldl=10, B=2, C=10, K=3, R=2, teacher_values=buf.data_ptr(), ldv=3, teacher_index=buf.data_ptr(), ldi=3,
                        temperature=T, alpha=1.0, grad_scale=1.0, loss_rows=buf.data_ptr())
    assert N.load().ep_distill_topk(C.byref(a), buf.data_ptr(), 1 << 20, 0) == -1


@pytest.mark.parametrize("tail", [False, True])
def test_a_rank_without_shards_has_a_teacher_too(tmp_path, tail):
    """More ranks than shards: every rank builds the same criterion; the empty one's table lists nothing."""
    w = TS.TokenStoreWriter(str(tmp_path), 2, 8, teacher_temperature=3.0)
    w.add(np.zeros((4, 2, 8)), np.zeros(4), teacher=(np.ones((4, 5)), np.ones((4, 5))) + ((np.ones(4),) if tail else ()))
    w.close()
    st = TS.ResidentTokenStore(str(tmp_path), "cpu", world=3, rank=2)
    assert st.num_images == 0 and st.num_batches(2) == 0
    crit = distill.TopKDistillation.from_store(st, alpha=0.5)
    assert crit.temperature == 3.0 and crit.teacher_values.shape == (1, 5) and (crit.teacher_index == -1).all() and (crit.teacher_tail is not None) == tail
    if tail:
        assert torch.isneginf(crit.teacher_tail).all()
