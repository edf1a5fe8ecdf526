"""Pre-dumped token store and feeder.

The reference can dump frozen-backbone tokens only as one small ``.npz`` (``tokens (n,N,C) float32``,
``images``, ``names``; reference tools/dump_tokens.py:95-98).  Training a probe on a 7B-parameter
encoder needs the whole dataset's tokens on disk once and then a reader that
keeps the head kernels fed.  This module provides

  * a sharded on-disk format: ``meta.json`` + ``tokens-XXXXX.bin`` (raw row-major ``(n_i, N, D)`` fp32 or bf16)
    + ``labels-XXXXX.npy``; shards are independent, so ranks partition them with no communication.  bf16 storage
    halves disk / HBM footprint (the 1.28 M x 196 x 4096 tokens of a ViT-7B fit 8 GPUs only in bf16); the token
    passes widen bf16 to fp32 on the fly and compute in fp32;
  * ``mxfp4`` storage (``mx4``): 4-bit codes in ``tokens-XXXXX.bin`` and their scales in ``scales-XXXXX.bin``, 17/32 byte per
    channel.  The writer quantises on the GPU; a resident store then holds an ``mx4.Mx4Tokens`` cache that the EP head's two token
    passes read in place.  Images of fewer tokens carry ``lengths-XXXXX.npy``;
  * a teacher's top logits beside the labels (any dtype of the tokens; ``teacher-XXXXX.npz`` with values / index / tail), which
    ``distill.TopKDistillation.from_store`` turns into the loss of a probe that learns from them;
  * ``TokenStoreWriter`` / ``read_reference_npz`` (imports the reference's ``.npz`` dump);
  * ``ResidentTokenStore``: a rank's shard loaded ONCE into HBM (288 GB per MI355X: 163 k images of
    256x768 fp32 tokens per GPU, the whole 1.28 M-image ImageNet train set on 8 GPUs) and batches
    drawn as an int32 index vector -- the pooling kernels read the selected images IN PLACE
    (``image_index`` of the C ABI), so an epoch never copies or re-uploads a token;
  * ``StreamingTokenLoader``: for stores larger than HBM, double-buffered pinned-host -> device
    copies on a side stream (PCIe-bound, ~80 k img/s at 256x768 fp32; see EXPERIMENTS.md section 3).
"""
from __future__ import annotations

import json
import os
from typing import Iterator, List, NamedTuple, Optional, Sequence, Tuple

import numpy as np
import torch

from . import mx4

META = "meta.json"


class TeacherRows(NamedTuple):
    """A teacher's K best logits of every image of a store (``distill.topk_distillation``); ``tail`` (or None) is the log mass of the
    classes behind them at ``temperature``."""
    values: torch.Tensor
    index: torch.Tensor
    tail: Optional[torch.Tensor]
    temperature: float


class TokenStoreWriter:
    def __init__(self, out_dir: str, num_tokens: int, dim: int, shard_images: int = 8192, dtype: str = "float32",
                 teacher_temperature: float = 1.0):
        if dtype not in ("float32", "bfloat16", "mxfp4"):
            raise NotImplementedError("token store dtype: float32, bfloat16 or mxfp4")
        if dtype == "bfloat16" and dim % 8 != 0:
            raise ValueError("bfloat16 token store: dim must be a multiple of 8")
        os.makedirs(out_dir, exist_ok=True)
        self.out_dir, self.N, self.D, self.shard_images, self.dtype = out_dir, num_tokens, dim, shard_images, dtype
        self.shards: List[dict] = []
        self._tok: List[np.ndarray] = []
        self._lab: List[np.ndarray] = []
        self._more: dict = {}                 # scales, lengths, teacher arrays: what some stores have beside tokens and labels
        self.teacher_temperature = float(teacher_temperature)
        self._n = 0

    def add(self, tokens, labels: np.ndarray, lengths=None, teacher=None) -> None:
        """``tokens`` (n, N, D): numpy, torch (any floating type, any device) or nested lists.  mxfp4: quantised on the GPU (a host array is copied there first), and ``lengths`` (n,)
        may give images fewer than N tokens.  ``teacher`` = (values (n, K), index (n, K)[, tail (n,)]) of ``distill.teacher_topk`` at
        this writer's ``teacher_temperature``.  Every ``add`` of a store brings the same parts."""
        if not isinstance(tokens, torch.Tensor):
            tokens = np.asarray(tokens)
        n, dims = len(tokens), tuple(tokens.shape)
        assert len(dims) == 3 and dims[1:] == (self.N, self.D), dims
        assert len(labels) == n
        if n == 0:
            return
        more = {}
        def host(t, dt):
            if isinstance(t, torch.Tensor):                    # (numpy has no bfloat16)
                t = (t.detach().float() if t.dtype == torch.bfloat16 else t.detach()).cpu().numpy()
            return np.ascontiguousarray(t, dtype=dt)
        if self.dtype == "mxfp4":
            x = torch.as_tensor(tokens).detach()
            cache = mx4.quantize_tokens(x if x.is_cuda else x.to("cuda"))
            tokens, more["scales"] = cache.codes.cpu().numpy(), cache.scales.cpu().numpy()
        else:
            tokens = host(tokens, np.float32)
            if lengths is not None:
                raise ValueError("images of fewer tokens are for mxfp4 stores")
        if lengths is not None:
            more["lengths"] = host(lengths, np.int32)
            if more["lengths"].shape != (n,) or more["lengths"].min() < 0 or more["lengths"].max() > self.N:
                raise ValueError(f"lengths must be ({n},) within [0, {self.N}]")
        if teacher is not None:
            if len(teacher) not in (2, 3):
                raise ValueError("teacher is (values, index) or (values, index, tail)")
            more["values"], index = host(teacher[0], np.float32), host(teacher[1], np.int64)
            if index.size and (index.min() < -2 ** 31 or index.max() >= 2 ** 31):
                raise ValueError("teacher classes must fit 32 bits")
            more["index"] = index.astype(np.int32)
            if len(teacher) == 3 and teacher[2] is not None:
                more["tail"] = host(teacher[2], np.float32)
            if more["values"].ndim != 2 or more["values"].shape != more["index"].shape or any(len(more[k]) != n for k in ("values", "index", "tail") if k in more):
                raise ValueError(f"teacher arrays must be ({n}, K), ({n}, K) and ({n},)")
        if (self.shards or self._n) and set(more) != set(self._more):
            raise ValueError(f"this store's images carry {sorted(self._more)}, these carry {sorted(more)}")
        if "values" in self._more and self._more["values"] and self._more["values"][0].shape[1] != more["values"].shape[1]:
            raise ValueError(f"this store's teacher rows have {self._more['values'][0].shape[1]} entries, these have {more['values'].shape[1]}")
        self._tok.append(tokens); self._lab.append(np.asarray(labels, dtype=np.int64)); self._n += n
        for k, v in more.items():
            self._more.setdefault(k, []).append(v)
        while self._n >= self.shard_images:
            self._flush(self.shard_images)

    def _flush(self, n: int) -> None:
        tok = np.concatenate(self._tok); lab = np.concatenate(self._lab)
        idx = len(self.shards)
        path = lambda name: os.path.join(self.out_dir, name)
        (tok[:n] if self.dtype == "mxfp4" else _encode(tok[:n], self.dtype)).tofile(path(f"tokens-{idx:05d}.bin"))
        np.save(path(f"labels-{idx:05d}.npy"), lab[:n])
        more = {k: np.concatenate(v) for k, v in self._more.items()}
        if "scales" in more:
            more["scales"][:n].tofile(path(f"scales-{idx:05d}.bin"))
        if "lengths" in more:
            np.save(path(f"lengths-{idx:05d}.npy"), more["lengths"][:n])
        if "values" in more:
            np.savez(path(f"teacher-{idx:05d}.npz"), **{k: more[k][:n] for k in ("values", "index", "tail") if k in more})
        self.shards.append({"index": idx, "images": int(n)})
        self._tok, self._lab, self._n = ([tok[n:]] if len(tok) > n else []), ([lab[n:]] if len(lab) > n else []), len(tok) - n
        self._more = {k: [v[n:]] for k, v in more.items()}          # (an empty rest keeps the widths for the next add)

    def close(self) -> dict:
        if self._n:
            self._flush(self._n)
        meta = {"format": "ep-token-store-v1", "num_tokens": self.N, "dim": self.D, "dtype": self.dtype,
                "shards": self.shards, "total_images": int(sum(s["images"] for s in self.shards))}
        if "lengths" in self._more:
            meta["lengths"] = True
        if "values" in self._more:
            meta["teacher"] = {"k": int(self._more["values"][0].shape[1]), "tail": "tail" in self._more, "temperature": self.teacher_temperature}
        with open(os.path.join(self.out_dir, META), "w") as f:
            json.dump(meta, f, indent=1)
        return meta


def _encode(tok: np.ndarray, dtype: str) -> np.ndarray:
    """fp32 -> stored element type; bf16 (round to nearest even) travels as its raw 16-bit pattern."""
    if dtype == "float32":
        return tok
    return torch.from_numpy(np.ascontiguousarray(tok)).to(torch.bfloat16).view(torch.int16).numpy()


def _to_torch(arr: np.ndarray, dtype: str) -> torch.Tensor:
    t = torch.from_numpy(np.ascontiguousarray(arr))
    return t.view(torch.bfloat16) if dtype == "bfloat16" else t


def read_reference_npz(path: str) -> Tuple[np.ndarray, List[str]]:
    """Tokens and names of a reference dump (tools/dump_tokens.py:95-98: keys tokens/images/names)."""
    z = np.load(path, allow_pickle=True)
    return np.asarray(z["tokens"], dtype=np.float32), [str(n) for n in z["names"]]


def load_meta(store_dir: str) -> dict:
    with open(os.path.join(store_dir, META)) as f:
        meta = json.load(f)
    if meta.get("format") != "ep-token-store-v1":
        raise ValueError(f"{store_dir}: not an ep token store")
    return meta


def shards_of_rank(meta: dict, world: int, rank: int) -> List[dict]:
    """Round-robin shard ownership: independent units, no data-path collective."""
    return [s for s in meta["shards"] if s["index"] % world == rank]


def steps_per_epoch(meta: dict, world: int, batch_size: int, per_shard: bool = False) -> int:
    """Batches EVERY rank yields per epoch: the minimum over the ranks of what each one's shards hold, computed from
    ``meta.json`` alone (no collective).  Whole shards are dealt round-robin, so ranks can own different image counts;
    every engine step ends in a blocking all-reduce of the flat gradients, so all ranks must run the same number of
    steps or the longer one hangs there.  The reference gets equal lengths from ``DistributedSampler`` (it pads by
    wrap-around, main_linprobe.py:286-287); here the surplus of the larger ranks is dropped, like ``drop_last``.
    ``per_shard``: batches never span shards (the streaming loader)."""
    counts = []
    for r in range(world):
        mine = shards_of_rank(meta, world, r)
        counts.append(sum(s["images"] // batch_size for s in mine) if per_shard
                      else sum(s["images"] for s in mine) // batch_size)
    return min(counts) if counts else 0


def open_shard(store_dir: str, meta: dict, shard: dict) -> Tuple[np.memmap, np.ndarray]:
    if meta.get("dtype") == "mxfp4":
        raise ValueError("a 4-bit store's shards hold codes and scales: open_shard_arrays")
    tok = np.memmap(os.path.join(store_dir, f"tokens-{shard['index']:05d}.bin"),
                    dtype=np.float32 if meta.get("dtype", "float32") == "float32" else np.int16, mode="r",
                    shape=(shard["images"], meta["num_tokens"], meta["dim"]))
    lab = np.load(os.path.join(store_dir, f"labels-{shard['index']:05d}.npy"))
    return tok, lab


def open_shard_arrays(store_dir: str, meta: dict, shard: dict) -> List[np.ndarray]:
    """What a shard stores of its tokens, one row per image: [tokens], or [codes, scales(, lengths)] of a 4-bit store."""
    if meta.get("dtype") != "mxfp4":
        return [open_shard(store_dir, meta, shard)[0]]
    path = lambda kind, ext: os.path.join(store_dir, f"{kind}-{shard['index']:05d}.{ext}")
    out = [np.memmap(path(kind, "bin"), dtype=np.uint8, mode="r", shape=(shard["images"], meta["num_tokens"], nb))
           for kind, nb in zip(("tokens", "scales"), mx4.row_bytes(meta["dim"]))]
    return out + ([np.load(path("lengths", "npy"))] if meta.get("lengths") else [])


def open_shard_labels(store_dir: str, shard: dict) -> np.ndarray:
    return np.load(os.path.join(store_dir, f"labels-{shard['index']:05d}.npy"))


def _buffers(meta: dict, images: int, device, pin: bool = False) -> List[torch.Tensor]:
    """Empty tensors for the arrays of ``open_shard_arrays``."""
    n, d = meta["num_tokens"], meta["dim"]
    dtype = meta.get("dtype", "float32")
    if dtype == "mxfp4":
        parts = [((images, n, nb), torch.uint8) for nb in mx4.row_bytes(d)] + ([((images,), torch.int32)] if meta.get("lengths") else [])
    else:
        parts = [((images, n, d), torch.float32 if dtype == "float32" else torch.bfloat16)]
    return [torch.empty(shape, dtype=dt, device=device, pin_memory=pin) for shape, dt in parts]


def _tokens(meta: dict, parts: List[torch.Tensor]):
    """The tensors of ``_buffers`` as what the heads take: a token tensor or an ``mx4.Mx4Tokens``."""
    if meta.get("dtype") != "mxfp4":
        return parts[0]
    return mx4.Mx4Tokens(parts[0], parts[1], meta["dim"], parts[2] if len(parts) > 2 else None)


class ResidentTokenStore:
    """This rank's shards, resident in HBM.  ``batches(batch_size, epoch)`` yields
    ``(store_tensor, image_index int32 (B,), targets int64 (B,))``: pass ``store_tensor`` as the tokens and
    ``image_index`` to ``ProbeHeadEngine.train_step`` -- no per-batch copy happens."""

    def __init__(self, store_dir: str, device, world: int = 1, rank: int = 0, seed: int = 0):
        meta = load_meta(store_dir)
        mine = shards_of_rank(meta, world, rank)
        n = sum(s["images"] for s in mine)
        self.meta, self.world = meta, world
        self.N, self.D, self.seed, self.rank = meta["num_tokens"], meta["dim"], seed, rank
        self.dtype = meta.get("dtype", "float32")
        parts = _buffers(meta, max(n, 1), device)
        if n == 0 and self.dtype == "mxfp4":                 # (a rank without shards: one image of zeros)
            for t in parts:
                t.zero_()
        labels, teacher = [], []
        off = 0
        for s in mine:
            for t, a in zip(parts, open_shard_arrays(store_dir, meta, s)):
                t[off:off + s["images"]].copy_(_to_torch(a, self.dtype))
            labels.append(open_shard_labels(store_dir, s)); off += s["images"]
            if meta.get("teacher"):
                teacher.append(np.load(os.path.join(store_dir, f"teacher-{s['index']:05d}.npz")))
        self.tokens = _tokens(meta, parts)
        self.num_images = n
        self.teacher: Optional[TeacherRows] = None
        if meta.get("teacher"):
            if not teacher:                                  # (a rank without shards: one row that lists nothing)
                k = meta["teacher"]["k"]
                teacher = [{"values": np.zeros((1, k), np.float32), "index": np.full((1, k), -1, np.int32), "tail": np.full(1, -np.inf, np.float32)}]
            cat = lambda k: torch.from_numpy(np.concatenate([t[k] for t in teacher])).to(device)
            self.teacher = TeacherRows(cat("values"), cat("index"), cat("tail") if meta["teacher"]["tail"] else None, meta["teacher"]["temperature"])
        self.labels = torch.from_numpy(np.concatenate(labels) if labels else np.zeros(0, np.int64)).to(device)

    @classmethod
    def from_tensors(cls, tokens, labels: torch.Tensor, seed: int = 0, teacher: Optional[TeacherRows] = None) -> "ResidentTokenStore":
        """A resident store around tokens that are already in HBM (synthetic benchmarks, tokens produced by a live encoder
        pass): ``tokens`` (n, N, D) fp32 / bf16 on the GPU or an ``mx4.Mx4Tokens`` cache, ``labels`` (n,) int64.  One rank's view
        (world = 1)."""
        if isinstance(tokens, mx4.Mx4Tokens) and tokens.image_index is not None:
            raise ValueError("a store holds a cache, not a batch of one")
        self = cls.__new__(cls)
        n, N, D = tokens.shape
        self.meta, self.world, self.N, self.D, self.seed, self.rank = {"num_tokens": N, "dim": D}, 1, N, D, seed, 0
        self.dtype = "mxfp4" if isinstance(tokens, mx4.Mx4Tokens) else "float32" if tokens.dtype == torch.float32 else "bfloat16"
        self.tokens, self.num_images, self.teacher = tokens, n, teacher
        self.labels = labels.to(device=tokens.device, dtype=torch.int64)
        return self

    def table(self, kind: str, eps: Optional[float] = None) -> torch.Tensor:
        """A per-token / per-image table over the WHOLE store, computed once and kept (indexed like ``tokens``, so a batch
        read in place through ``image_index`` finds its rows): functions of the frozen tokens alone, which the token passes
        of some heads would otherwise recompute from a third read of the batch in every step --
        ``"token_stats"``: (n, N, 2) {mean, rstd} of a LayerNorm over D with ``eps`` (CAE / JEPA / CaiT / CLIP / SimPool heads;
        the reference applies that LayerNorm to the tokens in every forward, e.g. poolings/cae/cae_att.py:104,
        poolings/simpool.py:52), ``"channel_stats"``: (n, 2, D) per-image column mean and sum of squared deviations (AIM's token
        BatchNorm, SimPool's mean-token query), ``"cbam_channel_table"``: (n, 3, D), ``"xhat_mean"``: (n, D) mean normalised token
        row (the CLIP head's query input; made from ``"token_stats"`` of the same ``eps``).  ``engine.attach_store(store)`` makes an
        engine look them up (``engine_finetune.train_one_epoch`` / ``evaluate`` do that for a ``StoreBatch``)."""
        from . import functional as F_
        if self.dtype == "mxfp4":
            raise ValueError("tables are of float32 / bfloat16 stores: a head that takes them reads a 4-bit store's batches decoded")
        key = (kind, None if eps is None else float(eps))
        cache = self.__dict__.setdefault("_tables", {})
        if key not in cache:
            fn = {"token_stats": lambda t, lo: F_.token_stats(t, eps), "channel_stats": lambda t, lo: F_.channel_stats(t),
                  "cbam_channel_table": lambda t, lo: F_.cbam_channel_table(t),
                  "xhat_mean": lambda t, lo: F_.token_xhat_mean(t, self.table("token_stats", eps)[lo:lo + t.shape[0]])}.get(kind)
            if fn is None:
                raise ValueError(f"unknown store table {kind!r}")
            n = self.tokens.shape[0]
            parts = [fn(self.tokens[lo:lo + 32768], lo) for lo in range(0, n, 32768)]  # bounded launch grids
            cache[key] = parts[0] if len(parts) == 1 else torch.cat(parts)
        return cache[key]

    def loader(self, batch_size: int, epoch: int = 0, shuffle: bool = True, drop_last: bool = True) -> "StoreEpoch":
        """One epoch as a sized iterable of ``StoreBatch(store_tensor, image_index, targets)`` -- what
        ``engine_finetune.train_one_epoch`` / ``evaluate`` take in place of a DataLoader (they need ``len()``)."""
        return StoreEpoch(self, batch_size, epoch, shuffle, drop_last)

    def num_batches(self, batch_size: int, drop_last: bool = True) -> int:
        """Batches per epoch.  Data parallel (world > 1): the same number on every rank (``steps_per_epoch``)."""
        if self.world > 1:
            return steps_per_epoch(self.meta, self.world, batch_size)
        return self.num_images // batch_size if drop_last else -(-self.num_images // batch_size)

    def batches(self, batch_size: int, epoch: int = 0, shuffle: bool = True, drop_last: bool = True):
        g = torch.Generator(device="cpu").manual_seed(self.seed * 1000003 + epoch * 101 + self.rank)
        order = torch.randperm(self.num_images, generator=g) if shuffle else torch.arange(self.num_images)
        order = order.to(dtype=torch.int32)
        if self.tokens.is_cuda:
            # through pinned memory, asynchronously: a copy from pageable memory blocks the host until the queue has drained
            # (one step latency per epoch -- visible when a store holds only a few batches); the host copy is kept until the
            # next epoch's replaces it
            self._order_host = order.pin_memory()
            order = self._order_host.to(self.tokens.device, non_blocking=True)
        if self.world > 1:                 # equal step counts on all ranks: each step all-reduces the gradients
            stop = self.num_batches(batch_size) * batch_size
        else:
            stop = self.num_images - (self.num_images % batch_size if drop_last else 0)
        labels = self.labels[order.long()]          # ONE gather per epoch: a batch is then two views, no kernel of its own
        for lo in range(0, stop, batch_size):
            yield StoreBatch(self.tokens, order[lo:lo + batch_size], labels[lo:lo + batch_size], owner=self)


class StoreBatch(tuple):
    """``(store_tensor, image_index, targets)``: a batch of a resident token store, read in place through the int32
    ``image_index``.  A type of its own so that ``engine_finetune.train_one_epoch`` / ``evaluate`` can tell it from a loader
    that yields ``(images, extra, target)`` -- for any other 3-tuple they keep the reference's ``batch[0]`` / ``batch[-1]``
    reading (reference engine_finetune.py:125-126,185-186)."""
    def __new__(cls, store, image_index, targets, owner=None):
        self = super().__new__(cls, (store, image_index, targets))
        self.owner = owner          # the ResidentTokenStore (its cached per-token / per-image tables: ``table()``), or None
        return self


class StoreEpoch:
    """``len()`` + iteration over one epoch of a ResidentTokenStore (see ``ResidentTokenStore.loader``)."""

    def __init__(self, store: ResidentTokenStore, batch_size: int, epoch: int, shuffle: bool, drop_last: bool):
        self.store, self.batch_size, self.epoch, self.shuffle, self.drop_last = store, batch_size, epoch, shuffle, drop_last

    def __len__(self) -> int:
        return self.store.num_batches(self.batch_size, self.drop_last)

    def __iter__(self):
        return self.store.batches(self.batch_size, self.epoch, self.shuffle, self.drop_last)


class StreamingTokenLoader:
    """Shards larger than HBM: memmap -> pinned staging -> device on a copy stream, two batches deep."""

    def __init__(self, store_dir: str, device, batch_size: int, world: int = 1, rank: int = 0):
        self.dir, self.device, self.B = store_dir, device, batch_size
        self.meta = load_meta(store_dir)
        self.shards = shards_of_rank(self.meta, world, rank)
        # data parallel: every rank stops after the same number of batches (see steps_per_epoch)
        self.limit = steps_per_epoch(self.meta, world, batch_size, per_shard=True) if world > 1 else None
        self.stream = torch.cuda.Stream(device=device)
        self.dtype = self.meta.get("dtype", "float32")
        self.stage = [_buffers(self.meta, batch_size, "cpu", pin=True) for _ in range(2)]
        self.dev = [_buffers(self.meta, batch_size, device) for _ in range(2)]

    def __len__(self):
        n = sum(s["images"] // self.B for s in self.shards)
        return n if self.limit is None else min(n, self.limit)

    def __iter__(self) -> Iterator[Tuple[torch.Tensor, torch.Tensor]]:
        k = 0
        pending = None
        copied = [None, None]     # H2D-complete events per buffer (host staging may be rewritten after them)
        consumed = [None, None]   # main-stream events: the consumer's kernels on a device buffer are enqueued before them
        main = torch.cuda.current_stream(self.device)
        total = len(self)
        for s in self.shards:
            if k >= total:
                break
            arrays, lab = open_shard_arrays(self.dir, self.meta, s), open_shard_labels(self.dir, s)
            for lo in range(0, s["images"] - self.B + 1, self.B):
                if k >= total:
                    break
                buf = k & 1
                if copied[buf] is not None:
                    copied[buf].synchronize()                     # previous H2D out of this staging buffer is done
                for t, a in zip(self.stage[buf], arrays):
                    t.copy_(_to_torch(a[lo:lo + self.B], self.dtype))
                with torch.cuda.stream(self.stream):
                    if consumed[buf] is not None:
                        self.stream.wait_event(consumed[buf])     # consumer finished with this device buffer
                    for t, h in zip(self.dev[buf], self.stage[buf]):
                        t.copy_(h, non_blocking=True)
                    ev = torch.cuda.Event(); ev.record(self.stream)
                copied[buf] = ev
                cur = (buf, torch.from_numpy(lab[lo:lo + self.B]).to(self.device), ev)
                if pending is not None:
                    main.wait_event(pending[2])
                    yield _tokens(self.meta, self.dev[pending[0]]), pending[1]
                    done = torch.cuda.Event(); done.record(main); consumed[pending[0]] = done
                pending = cur
                k += 1
        if pending is not None:
            main.wait_event(pending[2])
            yield _tokens(self.meta, self.dev[pending[0]]), pending[1]
