"""What the operators of a compact probe-training cache cost: tokens held in 4 bits (write, read back), attention pooling over
them (forward, forward + backward) and distillation from a teacher's top logits (forward, forward + gradient).

The 4-bit cache is the MX format of 32-value groups: E2M1 codes, two per byte with the even channel in the low nibble, and one
E8M0 scale byte per group (2^(byte-127); 255 = not a number).  A token row is padded to whole 128-channel blocks, so codes are
(M, N, Dp/2) uint8 and scales (M, N, Dp/32) uint8 with Dp = 128 * ceil(D/128).  The exponent of a group is
floor(log2(amax)) - 2, one more where amax >= 1.75 * 2^floor(log2(amax)); values round to the nearest code, ties to the even one.

``own`` false: the plain form (elementary torch operations in 32 bits).  ``own`` true: the calls a user of
``efficient_probing_amd`` makes.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _store(name, B, N, D, dtype):
    return {"name": name, "kind": "store", "B": B, "N": N, "D": D, "dtype": dtype}


def _pool(name, M, B, N, D, Q, per_image=False, ragged=False, train=False):
    """``M`` images in the cache, ``B`` of them in the batch (``M`` == ``B``: the batch is the cache)."""
    return {"name": name, "kind": "train" if train else "attend", "M": M, "B": B, "N": N, "D": D, "Q": Q, "per_image": per_image, "ragged": ragged}


def _distill(name, B, C, K, dtype, T, alpha, tail=False, rows=0, grad=True):
    """``rows`` > 0: the teacher's table holds that many images and the batch's rows of it are read through an index."""
    return {"name": name, "kind": "distill", "B": B, "C": C, "K": K, "dtype": dtype, "T": T, "alpha": alpha, "tail": tail, "rows": rows, "grad": grad}


def listed():
    return [
        # a token dump writes one small bf16 batch of a ViT-S encoder (196 patches + CLS) and a reader takes it back
        _store("store_vits_small", 8, 197, 384, "bf16"),
        # the dump of a ViT-B/14 encoder at the benchmark's 256 x 768 tokens, half its batch of 1024
        _store("store_vitb", 512, 256, 768, "fp32"),
        # one image answered alone: latency
        _pool("serve_one_image", 1, 1, 256, 768, 8),
        # evaluation on images of different sizes (ragged token counts, empty ones among them), picked from a resident store;
        # 1152 channels are SigLIP2 SO400M's
        _pool("eval_ragged_so400m", 1024, 512, 257, 1152, 12, ragged=True),
        # two long clips, per-clip queries: the token axis has to be split over the chip
        _pool("attend_long_clip", 2, 2, 50001, 1024, 16, per_image=True),
        # the benchmark's training batch, DINOv2 ViT-B/14 tokens, 8 queries
        _pool("train_vitb_q8", 1024, 1024, 256, 768, 8, train=True),
        # 32 queries (the reference's default) on ViT-L tokens
        _pool("train_vitl_q32", 256, 256, 196, 1024, 32, train=True),
        # ViT-7B tokens, the batch picked from the store through an index
        _pool("train_vit7b_q4", 256, 128, 196, 4096, 4, train=True),
        # the probe's training batch on ImageNet-1k classes, teacher's 32 best, half of the weight on the labels
        _distill("distill_in1k", 1024, 1000, 32, "fp32", 2.0, 0.5),
        # ImageNet-21k classes with the teacher's remaining mass, the teacher's rows read in place from the store's table
        _distill("distill_in21k_tail", 2048, 21841, 64, "bf16", 1.0, 1.0, tail=True, rows=8192),
        # few rows over a very long class axis
        _distill("distill_long_rows", 6, 131071, 128, "fp32", 4.0, 0.9, tail=True),
        # the loss alone, for one validation image
        _distill("distill_one_row", 1, 1000, 8, "fp16", 1.0, 1.0, grad=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "train", "train", "distill", "distill"])
    if kind == "distill":
        C = _log(rng, 2, 200000)
        B = min(_log(rng, 1, 4096), max(1, 40_000_000 // C))
        K = min(C, _log(rng, 1, 256))
        return _distill("", B, C, K, rng.choice(["fp32", "bf16", "fp16"]), rng.choice([0.5, 1.0, 2.0, 3.0, 4.0]), rng.choice([1.0, 0.9, 0.5]),
                        tail=K < C and rng.random() < 0.5, rows=rng.choice([0, 0, 2 * B + 3]), grad=rng.random() < 0.7)
    D = 64 * rng.randint(1, 24) if rng.random() < 0.7 else rng.choice([rng.randint(5, 700), 2048, 4096])
    if kind == "store":
        N = _log(rng, 1, 2000)
        B = min(_log(rng, 1, 2048), max(1, 80_000_000 // (N * D)))
        return _store("", B, N, D, rng.choice(["fp32", "bf16", "fp16"]))
    long = rng.random() < 0.3
    N = _log(rng, 2000, 60000) if long else _log(rng, 1, 1500)
    Q = rng.choice([1, 1, 4, 8, 12, 16, 32, rng.randint(1, 40)])
    B = min(_log(rng, 1, 4) if long else _log(rng, 1, 1024), max(1, int(1.5e9) // (N * D * max(Q, 8))))
    M = B if rng.random() < 0.5 else B + rng.randint(1, B)
    return _pool("", M, B, N, D, Q, per_image=rng.random() < 0.3, ragged=rng.random() < 0.4, train=kind == "train")


def work(case):
    k = case["kind"]
    if k == "store":
        n = case["B"] * case["N"] * case["D"]
        return {"bytes": n * ((4 if case["dtype"] == "fp32" else 2) + 17 / 32 + 2), "flops": 4 * n}
    if k in ("attend", "train"):
        tokens = case["B"] * case["N"] * (0.5 if case["ragged"] else 1.0)
        q = case["Q"] * case["D"] * 4
        rows = case["B"] * q
        queries = rows if case["per_image"] else q
        byte = tokens * case["D"] * 17 / 32 + queries + rows
        flop = 4 * tokens * case["D"] * case["Q"]
        if k == "train":  # dP in, dq out; dA = dP.x and dq = dS.x
            byte += rows + queries
            flop *= 2
        return {"bytes": byte, "flops": flop}
    e = 4 if case["dtype"] == "fp32" else 2
    n = case["B"] * case["C"]
    return {"bytes": n * e * (2 if case["grad"] else 1) + case["B"] * (case["K"] * 8 + 16), "flops": n * 8}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _tokens(shape, g):
    """Features as an encoder leaves them: channels of different spread and offset."""
    D = shape[-1]
    spread = torch.exp(0.5 * torch.randn(D, device=DEV, generator=g))
    return torch.randn(shape, device=DEV, generator=g) * spread + 0.2 * torch.randn(D, device=DEV, generator=g)


def _power(e):
    """2^e in float32, exact, for whole numbers -125 <= e <= 125."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _encode(x):
    """(..., D) float -> E2M1 values with their group exponents: (signed code values, exponent), padded to 128 channels."""
    D = x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, -D % 128))
    g = x.reshape(*x.shape[:-1], -1, 32)
    mant, ex = torch.frexp(g.abs().amax(-1))                   # amax = mant * 2^ex, mant in [0.5, 1)
    e = (ex - 3 + (mant >= 0.875).to(ex.dtype)).clamp(-125, 125)
    e = torch.where(mant > 0, e, torch.full_like(e, -125))
    v = g * _power(-e)[..., None]
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6.0)
    return torch.where(v < 0, -a, a), e


def _pack(val, e):
    """Code values and exponents -> (codes uint8, scales uint8)."""
    a = val.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(val) & (a > 0)).to(torch.uint8) * 8).reshape(*val.shape[:-2], -1)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _cache(M, N, D, g):
    codes = torch.empty((M, N, -(-D // 128) * 64), device=DEV, dtype=torch.uint8)
    scales = torch.empty((M, N, -(-D // 128) * 4), device=DEV, dtype=torch.uint8)
    step = max(1, 40_000_000 // (N * D))
    for lo in range(0, M, step):
        n = min(step, M - lo)
        codes[lo:lo + n], scales[lo:lo + n] = _pack(*_encode(_tokens((n, N, D), g)))
    return codes, scales


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    k = case["kind"]
    if k == "store":
        s["x"] = _tokens((case["B"], case["N"], case["D"]), g).to(DTYPES[case["dtype"]])
    elif k in ("attend", "train"):
        M, B, N, D, Q = case["M"], case["B"], case["N"], case["D"], case["Q"]
        s["codes"], s["scales"] = _cache(M, N, D, g)
        s["index"] = torch.randperm(M, device=DEV, generator=g)[:B].to(torch.int32) if M != B else None
        s["lengths"] = torch.randint(0, N + 1, (M,), device=DEV, generator=g, dtype=torch.int32) if case["ragged"] else None
        shape = (B, Q, D) if case["per_image"] else (Q, D)
        s["q"] = torch.randn(shape, device=DEV, generator=g) * 1.5      # scores of a trained head: a few units wide
        s["scale"] = D ** -0.5
        if k == "train":
            s["dP"] = torch.randn((B, Q, D), device=DEV, generator=g) / B
        if own:
            from efficient_probing_amd import mx4
            s["cache"] = mx4.Mx4Tokens(s["codes"], s["scales"], D, lengths=s["lengths"])
    else:
        B, C, K, T = case["B"], case["C"], case["K"], case["T"]
        R = case["rows"] or B
        s["logits"] = (2.0 * torch.randn((B, C), device=DEV, generator=g)).to(DTYPES[case["dtype"]])
        # the teacher: K distinct classes a row, its best logits descending, and the log-sum of exp(t/T) over all others
        stride = max(1, C // K)
        start = torch.randint(0, C, (R, 1), device=DEV, generator=g)
        order = torch.argsort(torch.rand((R, K), device=DEV, generator=g), dim=1)
        s["index"] = ((start + order * stride) % C).to(torch.int32)
        s["values"] = (6.0 + 3.0 * torch.randn((R, K), device=DEV, generator=g)).sort(dim=1, descending=True).values
        s["tail"] = torch.logsumexp(s["values"] / T, 1) - 0.5 - torch.rand((R,), device=DEV, generator=g) if case["tail"] else None
        s["rows"] = torch.randperm(R, device=DEV, generator=g)[:B].to(torch.int32) if case["rows"] else None
        s["targets"] = torch.randint(0, C, (B,), device=DEV, generator=g) if case["alpha"] < 1.0 else None
    return s


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _decode(codes, scales, D):
    lut = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    nib = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    val = lut[nib].reshape(*scales.shape, 32)
    mult = torch.where(scales == 255, math.nan, (scales.int() << 23).view(torch.float32))
    return (val * mult[..., None]).flatten(-2)[..., :D]


def _attend_plain(s):
    case = s["case"]
    codes, scales, lengths = s["codes"], s["scales"], s["lengths"]
    if s["index"] is not None:
        pick = s["index"].long()
        codes, scales = codes[pick], scales[pick]
        lengths = None if lengths is None else lengths[pick]
    x = _decode(codes, scales, case["D"])
    B, N, D = x.shape
    xt = x.transpose(1, 2).contiguous()
    q = s["q"] * s["scale"]
    S = torch.matmul(q, xt)                                             # (B, Q, N)
    if lengths is not None:
        keep = torch.arange(N, device=x.device)[None, None, :] < lengths[:, None, None]
        S = torch.where(keep, S, -math.inf)
        m = S.amax(-1, keepdim=True)
        p = torch.where(keep, torch.exp(S - torch.where(m == -math.inf, 0.0, m)), 0.0)
        l = p.sum(-1, keepdim=True)
        A = p / torch.where(l == 0, 1.0, l)
    else:
        p = torch.exp(S - S.amax(-1, keepdim=True))
        A = p / p.sum(-1, keepdim=True)
    P = torch.matmul(A, x)
    if case["kind"] == "attend":
        return P
    dP = s["dP"]
    dA = torch.matmul(dP, xt)
    dS = A * (dA - (dP * P).sum(-1, keepdim=True))
    dq = torch.matmul(dS, x) * s["scale"]
    return P, (dq if case["per_image"] else dq.sum(0))


def _distill_plain(s):
    """alpha T^2 KL(teacher || student at T) + (1 - alpha) cross-entropy, per row, and the gradient of its mean over rows.
    With a tail, every class that the teacher does not list is one more outcome on both sides."""
    case = s["case"]
    T, alpha = case["T"], case["alpha"]
    z = s["logits"].float()
    B, C = z.shape
    val, idx, tail = s["values"], s["index"].long(), s["tail"]
    if s["rows"] is not None:
        pick = s["rows"].long()
        val, idx = val[pick], idx[pick]
        tail = None if tail is None else tail[pick]
    t = val / T
    if tail is not None:
        t = torch.cat((t, tail[:, None]), 1)
    tm = t.amax(1, keepdim=True)
    te = torch.exp(t - tm)
    tl = tm + torch.log(te.sum(1, keepdim=True))
    p = torch.exp(t - tl)                                               # (B, K [+ 1])
    y = z / T
    m = y.amax(1, keepdim=True)
    e = torch.exp(y - m)
    lse = m + torch.log(e.sum(1, keepdim=True))
    lq = torch.gather(y, 1, idx) - lse
    if tail is not None:
        rest = e.scatter(1, idx, 0.0).sum(1, keepdim=True)
        lq = torch.cat((lq, m + torch.log(rest) - lse), 1)
    loss = alpha * T * T * torch.where(p > 0, p * (t - tl - lq), 0.0).sum(1)
    if alpha < 1.0:
        m1 = z.amax(1, keepdim=True)
        e1 = torch.exp(z - m1)
        s1 = e1.sum(1, keepdim=True)
        loss = loss + (1 - alpha) * ((m1 + torch.log(s1)) - torch.gather(z, 1, s["targets"][:, None]))[:, 0]
    if not case["grad"]:
        return loss
    soft = torch.exp(y - lse)
    if tail is not None:
        listed_ = torch.zeros_like(z).scatter(1, idx, 1.0)
        over = e / rest * p[:, -1:]                                     # the tail's share, spread as the student does
        grad = soft - torch.where(listed_ > 0, 0.0, over)
        grad = grad.scatter_add(1, idx, -p[:, :-1])
    else:
        grad = soft.scatter_add(1, idx, -p)
    grad = grad * (alpha * T / B)
    if alpha < 1.0:
        hard = e1 / s1
        hard = hard.scatter_add(1, s["targets"][:, None], torch.full((B, 1), -1.0, device=z.device))
        grad = grad + hard * ((1 - alpha) / B)
    return loss, grad.to(s["logits"].dtype)


def run(s):
    case = s["case"]
    k = case["kind"]
    if not own:
        if k == "store":
            val, e = _encode(s["x"])
            return (val * _power(e)[..., None]).flatten(-2)[..., :case["D"]].to(torch.bfloat16)
        return _distill_plain(s) if k == "distill" else _attend_plain(s)
    if k == "distill":
        from efficient_probing_amd import distill
        loss, grad = distill.topk_distillation(s["logits"], s["values"], s["index"], s["targets"], teacher_tail=s["tail"], teacher_rows=s["rows"],
                                               temperature=case["T"], alpha=case["alpha"], need_grad=case["grad"])
        return (loss, grad) if case["grad"] else loss
    from efficient_probing_amd import mx4
    if k == "store":
        return mx4.dequantize_tokens(mx4.quantize_tokens(s["x"]), dtype=torch.bfloat16)
    train = k == "train"
    P, S, ML = mx4.pool_forward(s["cache"], s["q"], s["scale"], per_image_queries=case["per_image"], image_index=s["index"], need_scores=train)
    if not train:
        return P
    dq = mx4.pool_backward(s["cache"], S, ML, s["dP"], s["scale"], P=P, per_image_queries=case["per_image"], image_index=s["index"])
    return P, dq


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_store(x):
    """Nearest representable value per group, found among all codes of the group's scale."""
    B, N, D = x.shape
    out = torch.empty((B, N, D), device=x.device, dtype=torch.float64)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=x.device, dtype=torch.float64)
    edge = (grid[1:] + grid[:-1]) / 2
    for b0 in range(0, B, max(1, 20_000_000 // (N * D))):
        b1 = min(B, b0 + max(1, 20_000_000 // (N * D)))
        for lo in range(0, D, 32):
            v = x[b0:b1, :, lo:lo + 32].double()
            top = v.abs().amax(-1, keepdim=True)
            power = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
            power = power + (torch.exp2(power + 1) <= top).double() - (torch.exp2(power) > top).double()
            base = torch.exp2(power)
            unit = torch.where(top >= 1.75 * base, base / 2, base / 4)
            a = v.abs() / unit
            low = torch.bucketize(a, edge, right=False)             # first edge >= a: a tie stays at the lower code ...
            tie = (low < 7) & (a == edge[low.clamp(max=6)]) & (low % 2 == 1)   # ... unless that one is odd
            out[b0:b1, :, lo:lo + 32] = torch.sign(v) * grid[low + tie.long()] * unit
    return out


def _exact_pool(s):
    case = s["case"]
    B, N, D, Q = case["B"], case["N"], case["D"], case["Q"]
    order = s["index"].tolist() if s["index"] is not None else range(B)
    lengths = s["lengths"].tolist() if s["lengths"] is not None else None
    mag = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], device=DEV, dtype=torch.float64) / 2
    train = case["kind"] == "train"
    P = torch.zeros((B, Q, D), device=DEV, dtype=torch.float64)
    dq = torch.zeros(s["q"].shape, device=DEV, dtype=torch.float64)
    for b, img in enumerate(order):
        n = N if lengths is None else lengths[img]
        if n == 0:
            continue
        c = s["codes"][img, :n].long()
        x = torch.empty((n, c.shape[1] * 2), device=DEV, dtype=torch.float64)
        for half, nib in ((0, c % 16), (1, c // 16)):
            x[:, half::2] = mag[nib % 8] * (1 - 2 * (nib // 8))
        x = (x * torch.pow(2.0, s["scales"][img, :n].double() - 127).repeat_interleave(32, 1))[:, :D]
        q = (s["q"][b] if case["per_image"] else s["q"]).double().requires_grad_(train)
        out = torch.softmax((q @ x.t()) * s["scale"], -1) @ x
        P[b] = out.detach()
        if train:
            gq, = torch.autograd.grad(out, q, s["dP"][b].double())
            if case["per_image"]:
                dq[b] = gq
            else:
                dq += gq
    return (P, dq) if train else P


def _exact_distill(s):
    case = s["case"]
    T, alpha = case["T"], case["alpha"]
    B, C = s["logits"].shape
    rows = s["rows"].long() if s["rows"] is not None else torch.arange(B, device=DEV)
    loss = torch.zeros(B, device=DEV, dtype=torch.float64)
    grad = torch.zeros((B, C), device=DEV, dtype=torch.float64)
    step = max(1, 20_000_000 // C)
    for lo in range(0, B, step):
        hi = min(B, lo + step)
        z = s["logits"][lo:hi].double().requires_grad_(True)
        r = rows[lo:hi]
        t = s["values"][r].double() / T
        idx = s["index"][r].long()
        logq = torch.log_softmax(z / T, 1)
        student = logq.gather(1, idx)
        if s["tail"] is not None:
            t = torch.cat((t, s["tail"][r].double()[:, None]), 1)
            seen = torch.zeros((hi - lo, C), device=DEV, dtype=torch.bool).scatter_(1, idx, True)
            student = torch.cat((student, torch.logsumexp(logq.masked_fill(seen, -math.inf), 1, keepdim=True)), 1)
        logp = torch.log_softmax(t, 1)
        terms = logp.exp() * (logp - student)
        row = alpha * T * T * terms.sum(1)
        if alpha < 1.0:
            row = row + (1 - alpha) * torch.nn.functional.cross_entropy(z, s["targets"][lo:hi], reduction="none")
        loss[lo:hi] = row.detach()
        if case["grad"]:
            grad[lo:hi], = torch.autograd.grad(row.sum() / B, z)
    return (loss, grad) if case["grad"] else loss


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "store":
        return _exact_store(s["x"])
    return _exact_distill(s) if case["kind"] == "distill" else _exact_pool(s)
