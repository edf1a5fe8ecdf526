"""Tokens held in 4 bits (MXFP4: E2M1 codes, one power-of-two scale per 32 channels) and the attention that reads them in place.

    cache = quantize_tokens(x)                                  # (B, N, D) fp32 / bf16 / fp16 -> Mx4Tokens
    x = dequantize_tokens(cache, image_index=idx)               # ... back, any images of it, as bf16 / fp32 / fp16
    P, S, ML = pool_forward(cache, queries, scale)              # functional.pool_forward with the cache in place of x
    dq = pool_backward(cache, S, ML, dP, scale, P=P)            # functional.pool_backward / pool_backward_per_image
    P = attention_pool(cache, queries, scale)                   # the two as one differentiable call
    y = pool_project(cache, queries, v_weight, scale)           # ... with the value projection: what EfficientProbing(cache) runs

A token costs 17/32 byte per channel instead of 4 (fp32) or 2 (bf16); the attention's two passes read just those bytes.  The
pooled vectors are those of the decoded values at fp32 accuracy (queries and gradients enter the products exactly down to 2^-11 of
the largest of their 32 channels, 2^-6 in rows of more than 1792 channels; of a smaller one at most 2^-35, 2^-30, of that largest is
lost); what 4 bits cost is decided when the tokens are written (11 - 13 % of their root mean square for Gaussian to
Laplace-distributed channels).  No CPU path; the reference has no
counterpart (its dump keeps float32 tokens, tools/dump_tokens.py:95-98).
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from . import functional as F_

GROUP = 32                 # channels that share a scale
BLOCK = 128                # a row is padded to whole blocks of 128 channels
MAX_DIM = 4096             # widest row the attention takes
_OUT = {torch.float32: N.EP_DTYPE_F32, torch.bfloat16: N.EP_DTYPE_BF16, torch.float16: N.EP_DTYPE_F16}


def row_bytes(dim: int) -> Tuple[int, int]:
    """(code bytes, scale bytes) of one token."""
    blocks = -(-dim // BLOCK)
    return blocks * 64, blocks * 4


def _check_index(t: torch.Tensor, name: str, n: Optional[int]) -> None:
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or (n is not None and t.shape[0] != n) or t.shape[0] < 1:
        raise ValueError(f"{name} must be a contiguous int32 vector" + (f" of {n}" if n else ""))


class Mx4Tokens:
    """``codes`` (M, N, Dp/2) and ``scales`` (M, N, Dp/32) uint8 with Dp = ``dim`` rounded up to 128; ``lengths`` (M,) int32 gives
    images fewer than N tokens (whatever their other rows hold is masked out of the attention).  ``image_index`` (B,) int32
    makes it a BATCH: image b is cache image ``image_index[b]``, read in place.

    Codes count through the E2M1 grid 0, 0.5, 1, 1.5, 2, 3, 4, 6 (bit 3: sign), the even channel in the low nibble; a scale byte s
    stands for 2^(s - 127), 255 for a group that is not a number.  Pad channels hold code 0 and a finite scale."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, dim: int, lengths: Optional[torch.Tensor] = None,
                 image_index: Optional[torch.Tensor] = None):
        if codes.dim() != 3 or scales.dim() != 3 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError(f"codes and scales must be (M, N, bytes) uint8, got {tuple(codes.shape)} {codes.dtype} and {tuple(scales.shape)} {scales.dtype}")
        if dim < 1 or codes.shape[:2] != scales.shape[:2] or (codes.shape[2], scales.shape[2]) != row_bytes(dim):
            raise ValueError(f"{dim} channels take rows of {row_bytes(dim)} code / scale bytes, got {tuple(codes.shape)} and {tuple(scales.shape)}")
        if codes.shape[0] < 1 or codes.shape[1] < 1:
            raise ValueError(f"an empty cache: {tuple(codes.shape)}")
        for t, name in ((codes, "codes"), (scales, "scales")):
            if t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != t.shape[2]) or (t.shape[0] > 1 and t.stride(0) < t.shape[1] * t.shape[2]):
                raise ValueError(f"{name}: the rows of an image must be contiguous and images must not overlap (strides {t.stride()})")
        for t, name, n in ((lengths, "lengths", codes.shape[0]), (image_index, "image_index", None)):
            if t is not None:
                _check_index(t, name, n)
        devices = {t.device for t in (codes, scales, lengths, image_index) if t is not None}
        if len(devices) != 1:
            raise ValueError(f"codes, scales, lengths and image_index must be on one device, got {sorted(map(str, devices))}")
        self.codes, self.scales, self.dim, self.lengths, self.image_index = codes, scales, int(dim), lengths, image_index

    @classmethod
    def _made(cls, codes, scales, dim, lengths, image_index=None) -> "Mx4Tokens":
        """Around tensors that are known to fit (5 us of checks less per call)."""
        self = cls.__new__(cls)
        self.codes, self.scales, self.dim, self.lengths, self.image_index = codes, scales, dim, lengths, image_index
        return self

    # -- what the loops look at in a token tensor
    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def is_cuda(self) -> bool:
        return self.codes.is_cuda

    @property
    def shape(self) -> torch.Size:
        """(B, N, D) of the batch this stands for."""
        b = self.codes.shape[0] if self.image_index is None else self.image_index.shape[0]
        return torch.Size((b, self.codes.shape[1], self.dim))

    @property
    def nbytes(self) -> int:
        return self.codes.shape[0] * self.codes.shape[1] * sum(row_bytes(self.dim))

    def __len__(self) -> int:
        return self.shape[0]

    def select(self, image_index: torch.Tensor) -> "Mx4Tokens":
        """The batch of these images (no copy)."""
        if self.image_index is not None:
            raise ValueError("this is a batch of a cache already: select from the cache")
        _check_index(image_index, "image_index", None)
        if image_index.device != self.codes.device:
            raise ValueError(f"image_index is on {image_index.device}, the cache on {self.codes.device}")
        return self._made(self.codes, self.scales, self.dim, self.lengths, image_index)

    def images(self, lo: int, hi: int) -> "Mx4Tokens":
        """Images lo .. hi - 1 (a view; what a writer fills in ranges)."""
        if self.image_index is not None or not 0 <= lo < hi <= self.codes.shape[0]:
            raise ValueError(f"images {lo} .. {hi} of a cache of {self.codes.shape[0]}" if self.image_index is None else "images() is for a cache, not a batch")
        return Mx4Tokens(self.codes[lo:hi], self.scales[lo:hi], self.dim, None if self.lengths is None else self.lengths[lo:hi])

    def tokens(self, lo: int, hi: int) -> "Mx4Tokens":
        """Tokens lo .. hi - 1 of every image (a view, such as ``tokens(1, N)`` without [CLS]); lengths shrink with it."""
        if not 0 <= lo < hi <= self.codes.shape[1]:
            raise ValueError(f"tokens {lo} .. {hi} of rows of {self.codes.shape[1]}")
        ln = None if self.lengths is None else (self.lengths - lo).clamp_(0, hi - lo)
        return Mx4Tokens(self.codes[:, lo:hi], self.scales[:, lo:hi], self.dim, ln, self.image_index)

    def to(self, device, non_blocking: bool = False) -> "Mx4Tokens":
        if torch.device(device) == self.device or (torch.device(device).type == self.device.type and torch.device(device).index is None):
            return self
        mv = lambda t: None if t is None else t.to(device, non_blocking=non_blocking)
        return Mx4Tokens(mv(self.codes), mv(self.scales), self.dim, mv(self.lengths), mv(self.image_index))

    def _parts(self) -> Tuple[Optional[torch.Tensor], ...]:
        return self.codes, self.scales, self.lengths, self.image_index

    def _versions(self) -> Tuple[Optional[int], ...]:
        """What changes when any of the tensors is written (those of inference mode keep no count)."""
        return tuple(None if t is None or t.is_inference() else t._version for t in self._parts())

    def _args(self, image_index: Optional[torch.Tensor] = None) -> "N.EPMx4Tokens":
        codes = self.codes
        N.require_gpu_tensor(codes, "codes")
        M, n, _ = codes.shape
        idx = self.image_index
        if image_index is not None:
            if idx is not None:
                raise ValueError("this is a batch of a cache already: select from the cache")
            _check_index(image_index, "image_index", None)
            idx = image_index
        return N.EPMx4Tokens(codes.data_ptr(), self.scales.data_ptr(), codes.stride(0), self.scales.stride(0), F_._ptr(self.lengths),
                             F_._ptr(idx), M, M if idx is None else idx.shape[0], n, self.dim)


def empty_cache(images: int, num_tokens: int, dim: int, device, lengths: Optional[torch.Tensor] = None) -> Mx4Tokens:
    """A cache to be written range by range: ``quantize_tokens(x, out=cache.images(lo, hi))``."""
    cb, sb = row_bytes(dim)
    codes = torch.empty((images, num_tokens, cb), device=device, dtype=torch.uint8)
    scales = torch.empty((images, num_tokens, sb), device=device, dtype=torch.uint8)
    if lengths is None and images > 0 and num_tokens > 0 and dim > 0:
        return Mx4Tokens._made(codes, scales, int(dim), None)
    return Mx4Tokens(codes, scales, dim, lengths)


def _on(t: torch.Tensor, *others: Optional[torch.Tensor]) -> torch.device:
    for o in others:
        if o is not None and o.device != t.device:
            raise ValueError(f"tensors on {t.device} and {o.device}")
    return t.device


def quantize_tokens(x: torch.Tensor, out: Optional[Mx4Tokens] = None, lengths: Optional[torch.Tensor] = None) -> Mx4Tokens:
    """(B, N, D) tokens -> a cache of B images, or into ``out`` (a cache or a range of one, of the same shape; its ``lengths`` stay).
    Any strides over images and tokens are read in place.  A group of 32 channels that holds a NaN or an infinity becomes NaN."""
    N.require_gpu_tensor(x, "tokens")
    if x.dim() != 3 or min(x.shape) < 1:
        raise ValueError(f"tokens must be (B, N, D), got {tuple(x.shape)}")
    B, n, D = x.shape
    if x.dtype not in _OUT:
        x = x.float()
    if x.stride(2) != 1 or min(x.stride()) < 0:
        x = x.contiguous()
    given = out is not None
    if not given:
        out = empty_cache(B, n, D, x.device, lengths)
    elif lengths is not None:
        raise ValueError("lengths belong to a new cache; `out` has its own")
    if tuple(out.shape) != (B, n, D) or out.image_index is not None:
        raise ValueError(f"out must be a cache of {(B, n, D)}, got {tuple(out.shape)}" + (" as a batch" if out.image_index is not None else ""))
    with N.device_guard(_on(x, out.codes)):
        N.check(N.load().ep_mx4_quantize(x.data_ptr(), _OUT[x.dtype], x.stride(0), x.stride(1), B, n, D, out.codes.data_ptr(),
                                         out.scales.data_ptr(), out.codes.stride(0), out.scales.stride(0),
                                         N.current_stream_ptr(x.device)), "ep_mx4_quantize")
    if given:                                                   # (the kernel's writes are not seen by torch's own count)
        torch.autograd.graph.increment_version((out.codes, out.scales))
    return out


def dequantize_tokens(cache: Mx4Tokens, dtype: torch.dtype = torch.bfloat16, image_index: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The batch's tokens (B, N, D) as ``dtype``: exact in bf16 and fp32, rounded in fp16.  Every row is read back, also those behind
    an image's length; an index outside the cache gives NaN."""
    if dtype not in _OUT:
        raise ValueError(f"dtype must be one of {sorted(map(str, _OUT))}, got {dtype}")
    args = cache._args(image_index)
    out = torch.empty((args.B, args.N, args.D), device=cache.device, dtype=dtype)
    with N.device_guard(_on(out, image_index)):
        N.check(N.load().ep_mx4_dequantize(C.byref(args), out.data_ptr(), _OUT[dtype], N.current_stream_ptr(out.device)), "ep_mx4_dequantize")
    return out


def _queries(cache: Mx4Tokens, queries: torch.Tensor, per_image: bool, B: int) -> Tuple[torch.Tensor, int]:
    q = F_._f32c(queries, "queries")
    D = cache.dim
    ok = tuple(q.shape) == (B, q.shape[-2], D) if per_image and q.dim() == 3 else (not per_image and q.dim() in (2, 3) and q.shape[-1] == D and q.numel() == q.shape[-2] * D)
    if not ok or q.shape[-2] < 1:
        want = f"({B}, Q, {D})" if per_image else f"(Q, {D}) or (1, Q, {D})"
        raise ValueError(f"queries must be {want}, got {tuple(queries.shape)}")
    if D > MAX_DIM:
        raise ValueError(f"the attention over a 4-bit cache takes at most {MAX_DIM} channels, got {D}")
    return _aligned(q), q.shape[-2]


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """16-byte aligned storage, as the kernels read operand rows."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _padded(n: int) -> int:
    """Row stride of saved scores: whole 16-byte pieces."""
    return (n + 3) // 4 * 4


@functools.lru_cache(maxsize=256)
def _workspace_bytes(B: int, n: int, D: int, Q: int, device: int) -> int:
    return N.load().ep_mx4_pool_workspace_bytes(B, n, D, Q)


def _workspace(B: int, n: int, D: int, Q: int, device) -> Tuple[Optional[torch.Tensor], int]:
    """(scratch or None, bytes); to be called with ``device`` current: its compute units decide how the work is cut."""
    nbytes = _workspace_bytes(B, n, D, Q, device.index)
    return (torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None), nbytes


def pool_forward(cache: Mx4Tokens, queries: torch.Tensor, scale: float, per_image_queries: bool = False,
                 image_index: Optional[torch.Tensor] = None, need_scores: bool = True):
    """``functional.pool_forward`` over a 4-bit cache: P (B, Q, D), S (B, Q, N) or None without ``need_scores``, ML (B, Q, 4) with the
    row maximum and the sum of exponentials (S is a view of rows padded to a multiple of 4).  ``queries`` (Q, D) / (1, Q, D), or (B, Q, D) with ``per_image_queries``.  Tokens behind an
    image's length have score -inf; an image without tokens pools to 0; an index outside the cache gives NaN."""
    args = cache._args(image_index)
    B, n, D = args.B, args.N, args.D
    q, Q = _queries(cache, queries, per_image_queries, B)
    dev = _on(cache.codes, q, image_index)
    P = q.new_empty((B, Q, D))
    S = q.new_empty((B, Q, _padded(n)))[:, :, :n] if need_scores else None
    ML = q.new_empty((B, Q, 4))
    with N.device_guard(dev):
        ws, nbytes = _workspace(B, n, D, Q, dev)
        N.check(N.load().ep_mx4_pool_forward(C.byref(args), q.data_ptr(), Q * D if per_image_queries else 0, Q, float(scale), P.data_ptr(),
                                             F_._ptr(S), _padded(n), ML.data_ptr(), F_._ptr(ws), nbytes, N.current_stream_ptr(dev)), "ep_mx4_pool_forward")
    return P, S, ML


def pool_backward(cache: Mx4Tokens, S: torch.Tensor, ML: torch.Tensor, dP: torch.Tensor, scale: float, P: Optional[torch.Tensor] = None,
                  per_image_queries: bool = False, image_index: Optional[torch.Tensor] = None, dq: Optional[torch.Tensor] = None,
                  accumulate: bool = False) -> torch.Tensor:
    """Gradient of the query rows from dP: (Q, D) summed over the batch (in a fixed order), or (B, Q, D) with ``per_image_queries``.
    delta = dP . P comes from ``P`` when given, else from ``ML[..., 2]`` (``functional.project_backward`` leaves it there).  An image
    without tokens, or an index outside the cache, adds nothing."""
    args = cache._args(image_index)
    B, n, D = args.B, args.N, args.D
    Q = S.shape[1] if S.dim() == 3 else -1
    dP = _aligned(F_._f32c(dP, "dP"))
    P = None if P is None else _aligned(P)
    if tuple(S.shape) != (B, Q, n) or S.dtype != torch.float32:
        raise ValueError(f"S must be float32 {(B, Q, n)}, got {tuple(S.shape)} {S.dtype}")
    if S.stride(2) != 1 or S.stride(1) % 4 or S.stride(1) < n or S.stride(0) != Q * S.stride(1) or S.data_ptr() % 16:
        S = torch.nn.functional.pad(S, (0, _padded(n) - n)).contiguous()      # not as pool_forward left it
    for t, name, shape in ((ML, "ML", (B, Q, 4)), (dP, "dP", (B, Q, D)), (P, "P", (B, Q, D))):
        if t is not None and (tuple(t.shape) != shape or t.dtype != torch.float32 or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous float32 {shape}, got {tuple(t.shape)} {t.dtype}")
    if D > MAX_DIM:
        raise ValueError(f"the attention over a 4-bit cache takes at most {MAX_DIM} channels, got {D}")
    shape = (B, Q, D) if per_image_queries else (Q, D)
    if dq is None:
        if accumulate:
            raise ValueError("accumulate needs dq")
        dq = torch.empty(shape, device=dP.device, dtype=torch.float32)
    elif tuple(dq.shape) != shape or dq.dtype != torch.float32 or not dq.is_contiguous():
        raise ValueError(f"dq must be contiguous float32 {shape}, got {tuple(dq.shape)} {dq.dtype}")
    if accumulate and per_image_queries:
        raise ValueError("accumulate is for shared queries")
    dev = _on(cache.codes, S, ML, dP, P, dq, image_index)
    with N.device_guard(dev):
        ws, nbytes = _workspace(B, n, D, Q, dev)
        N.check(N.load().ep_mx4_pool_backward(C.byref(args), Q, float(scale), S.data_ptr(), S.stride(1), ML.data_ptr(), F_._ptr(P), dP.data_ptr(),
                                              dq.data_ptr(), int(per_image_queries), int(accumulate), F_._ptr(ws), nbytes,
                                              N.current_stream_ptr(dev)), "ep_mx4_pool_backward")
    return dq


def attention(cache: Mx4Tokens, queries: torch.Tensor, scale: float, per_image_queries: bool = False,
              image_index: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale * queries . x) over the tokens, (B, Q, N): 0 behind an image's length (everywhere for one without tokens)."""
    _, S, ML = pool_forward(cache, queries, scale, per_image_queries, image_index)
    return F_.attention_from_scores(S.contiguous(), ML).masked_fill_(ML[..., 1:2] == 0, 0.0)


def _keep_cache(ctx, cache: Mx4Tokens) -> None:
    """For the backward pass, with the versions that its tensors have now."""
    ctx.cache, ctx.versions = Mx4Tokens._made(cache.codes, cache.scales, cache.dim, cache.lengths, cache.image_index), cache._versions()


def _kept_cache(ctx) -> Mx4Tokens:
    if ctx.cache._versions() != ctx.versions:
        raise RuntimeError("one of the 4-bit cache's tensors needed for gradient computation has been modified since the forward pass "
                           "(quantize_tokens(out=...) or an in-place operation)")
    return ctx.cache


class _AttentionPool(torch.autograd.Function):
    @staticmethod
    def forward(ctx, queries, cache, scale, per_image):
        need = ctx.needs_input_grad[0]
        P, S, ML = pool_forward(cache, queries, scale, per_image, need_scores=need)
        if need:
            ctx.save_for_backward(P, S, ML)
        _keep_cache(ctx, cache)
        ctx.scale, ctx.per_image, ctx.qshape = scale, per_image, queries.shape
        return P

    @staticmethod
    @once_differentiable
    def backward(ctx, dP):
        P, S, ML = ctx.saved_tensors
        dq = pool_backward(_kept_cache(ctx), S, ML, dP, ctx.scale, P=P, per_image_queries=ctx.per_image)
        return dq.reshape(ctx.qshape), None, None, None


def attention_pool(cache: Mx4Tokens, queries: torch.Tensor, scale: float, per_image_queries: bool = False,
                   image_index: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale * queries . x) x over the cache's tokens, differentiable in ``queries`` (the tokens are frozen): (B, Q, D).  The
    backward pass reads the cache again: one that was written in between is an error."""
    if image_index is not None:
        cache = cache.select(image_index)
    return _AttentionPool.apply(queries, cache, float(scale), per_image_queries)


class _PoolProject(torch.autograd.Function):
    """``functional.ep_pool_project`` over a 4-bit cache."""

    @staticmethod
    def forward(ctx, queries, v_weight, cache, scale, per_image):
        need = ctx.needs_input_grad[0]
        P, S, ML = pool_forward(cache, queries, scale, per_image, need_scores=need)
        y = F_.project_forward(P, v_weight)
        ctx.save_for_backward(P, S, ML, y, v_weight)
        _keep_cache(ctx, cache)
        ctx.scale, ctx.per_image, ctx.qshape = scale, per_image, queries.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        P, S, ML, y, v_weight = ctx.saved_tensors
        need_q = ctx.needs_input_grad[0]
        dP, dWv = F_.project_backward(dy.contiguous(), y, P, v_weight, None, need_dP=need_q, need_dWv=ctx.needs_input_grad[1])
        dq = pool_backward(_kept_cache(ctx), S, ML, dP, ctx.scale, P=P, per_image_queries=ctx.per_image).reshape(ctx.qshape) if need_q else None
        return dq, dWv, None, None, None


def pool_project(cache: Mx4Tokens, queries: torch.Tensor, v_weight: torch.Tensor, scale: float, per_image_queries: bool = False) -> torch.Tensor:
    """``attention_pool``, then the value projection of each query's slice: (B, D') with D' = v_weight.shape[0]."""
    return _PoolProject.apply(queries, v_weight, cache, float(scale), per_image_queries)
