"""Operators of a language model's training step: what is timed and compared.

`listed()` names the cases, `draw(rng)` gives further ones of the same ranges, `prepare` makes
what a program holds before the call, `run` makes one pass (in plain torch operations, or with
`own` through this package), `exact` is the same function in float64.  Four operators:

  ce        linear_cross_entropy: softmax cross entropy of hidden rows against a head matrix;
            loss, and in training the gradients of the rows and of the matrix
  embed     embedding: rows of a table, scaled; in training the table's gradient
  balance   balance_loss: per-expert counts, the load-balance loss and its gradient
  clip      clip_grads: the global norm of many gradients, and the clipped gradients

All inputs are made on the GPU from the seed."""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
VOCAB = 100277  # the language model's vocabulary and width
WIDTH = 1024


def _ce(tokens, **kw):
    return dict(dict(op="ce", tokens=tokens, d=WIDTH, vocab=VOCAB, dtype="bf16", train=True, ignored=0.0, reduction="mean"), **kw)


def _embed(tokens, **kw):
    return dict(dict(op="embed", tokens=tokens, d=WIDTH, vocab=VOCAB, dtype="bf16", train=True, scale=1.0, padding=-1, zipf=1.0), **kw)


def _balance(tokens, **kw):
    return dict(dict(op="balance", tokens=tokens, heads=8, top_k=16, experts=262144, dtype="fp32", zipf=0.0), **kw)


def _clip(blocks, **kw):
    return dict(dict(op="clip", blocks=blocks, d=WIDTH, vocab=VOCAB, experts=262144, dtype="bf16", norm=2.0, share=0.5), **kw)


def listed():
    return [
        # the loss of a training batch: two sequences of 2,048 tokens, every position counts
        dict(_ce(4096), name="ce_train_4096"),
        # instruction tuning: an odd number of tokens, two thirds of them prompt, which has no label
        dict(_ce(1777, ignored=0.66), name="ce_train_1777_masked"),
        # validation: the loss of every token of four sequences of 2,048, no gradients
        dict(_ce(8192, train=False, reduction="none"), name="ce_score_8192"),
        # scoring one short answer
        dict(_ce(7, train=False, reduction="sum"), name="ce_score_7"),
        # a small float32 model's training batch, odd sizes
        dict(_ce(500, d=256, vocab=8009, dtype="fp32"), name="ce_train_fp32_500"),
        # the embedding of a training batch of 8,192 tokens with a natural skew, and its gradient
        dict(_embed(8192), name="embed_train_8192"),
        # a decode step of 64 sequences, rows scaled by sqrt(d)
        dict(_embed(64, train=False, scale=32.0), name="embed_decode_64"),
        # a small float32 table of odd width, half of the batch padding
        dict(_embed(1500, d=101, vocab=5003, dtype="fp32", scale=0.5, padding=0), name="embed_train_fp32_1500"),
        # the balance of a training batch over 262,144 experts
        dict(_balance(4096), name="balance_4096"),
        # a short batch with skewed experts, gates in bfloat16
        dict(_balance(500, heads=4, top_k=8, experts=4096, dtype="bf16", zipf=1.1), name="balance_500_skewed"),
        # clipping the gradients of a model of four expert blocks, some 300 MB of latents among 160 tensors
        dict(_clip(4), name="clip_4_blocks"),
        # clipping a small float32 model's gradients: many small tensors
        dict(_clip(3, d=64, vocab=500, experts=256, dtype="fp32"), name="clip_small"),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ce", "ce", "ce", "ce", "ce_fp32", "embed", "embed", "balance", "balance", "clip"])
    if op == "ce":
        train = rng.random() < 0.6
        return _ce(_log(rng, 1, 4096 if train else 8192), d=8 * _log(rng, 8, 128), vocab=_log(rng, 500, VOCAB), train=train,
                   ignored=rng.choice([0.0, 0.0, 0.1, 0.5, 0.9]), reduction=rng.choice(["mean", "sum", "none"]))
    if op == "ce_fp32":
        return _ce(_log(rng, 1, 1000), d=8 * _log(rng, 4, 64), vocab=_log(rng, 300, 20000), dtype="fp32", train=rng.random() < 0.7,
                   ignored=rng.choice([0.0, 0.3]), reduction=rng.choice(["mean", "sum", "none"]))
    if op == "embed":
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        return _embed(_log(rng, 1, 8192), d=_log(rng, 32, 1024), vocab=_log(rng, 500, VOCAB), dtype=dtype, train=rng.random() < 0.7,
                      scale=rng.choice([1.0, 0.5, 27.7]), padding=rng.choice([-1, -1, 0, 17]), zipf=rng.choice([0.0, 1.0, 1.3]))
    if op == "balance":
        return _balance(_log(rng, 1, 4096), heads=rng.choice([2, 4, 8]), top_k=rng.choice([4, 8, 16]),
                        experts=_log(rng, 16, 512) ** 2, dtype=rng.choice(["fp32", "bf16"]), zipf=rng.choice([0.0, 0.8, 1.1]))
    return _clip(rng.randint(1, 4), d=rng.choice([64, 200, 512, 1024]), vocab=_log(rng, 500, VOCAB), experts=_log(rng, 16, 512) ** 2,
                 dtype=rng.choice(["bf16", "fp32"]), norm=rng.choice([2.0, 2.0, math.inf]), share=rng.choice([0.1, 0.5, 2.0])) \
        if rng.random() < 0.5 else _clip(rng.randint(1, 4), d=64, vocab=500, experts=256, dtype="fp32")


# ------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _ids(g, shape, n, zipf):
    """Whole numbers below n: uniform, or with frequencies (rank + 1)^-zipf."""
    if zipf == 0.0:
        return torch.randint(0, n, shape, generator=g, device=DEV)
    w = (torch.arange(n, device=DEV, dtype=torch.float64) + 1.0) ** -zipf
    cdf = torch.cumsum(w, 0)
    u = torch.rand(shape, generator=g, device=DEV, dtype=torch.float64) * cdf[-1]
    return torch.searchsorted(cdf, u).clamp_(max=n - 1)


def _clip_shapes(c):
    """The shapes of the parameters of a model of `blocks` expert blocks."""
    d, E = c["d"], c["experts"]
    K = math.isqrt(E)
    shapes = [(c["vocab"], d), (d,)]
    for _ in range(c["blocks"]):
        shapes += [(E, 128), (512, 128), (2 * d, 512), (K, 128), (K, 128)]
        for _ in range(8):
            shapes += [(256, d), (256,), (256,), (256,)]
        q, kv = d * 3 // 4, d // 4
        shapes += [(q, d), (q,), (2 * d, q), (kv + 64, d), (kv,), (2 * d, kv), (d, d), (d,), (d,)]
    return shapes


def prepare(case, seed):
    g = _gen(seed)
    c, dt = case, DTYPES[case["dtype"]]
    st = {"case": case}
    rn = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    if c["op"] == "ce":
        n, d, V = c["tokens"], c["d"], c["vocab"]
        w = rn(V, d) * 0.05
        labels = _ids(g, (n,), V, 1.0)
        # rows lean to their label's row, as a trained model's do
        h = rn(n, d) + w[labels] * (rn(n, 1).abs() * 2.0 * math.sqrt(1024 / d))
        if c["ignored"] > 0.0:
            # runs of unlabelled positions, as prompts and padding are
            runs = (torch.arange(n, device=DEV) + torch.randint(0, 64, (1,), generator=g, device=DEV)) // 64
            off = torch.rand(int(runs[-1]) + 1, generator=g, device=DEV) < c["ignored"]
            off[0] = False
            labels = torch.where(off[runs], torch.full_like(labels, -100), labels)
        st.update(h=h.to(dt).requires_grad_(c["train"]), w=w.to(dt).requires_grad_(c["train"]), labels=labels)
        if c["train"]:
            st["gy"] = rn(n).abs() / n if c["reduction"] == "none" else torch.ones((), device=DEV)
    elif c["op"] == "embed":
        n, d, V = c["tokens"], c["d"], c["vocab"]
        ids = _ids(g, (n,), V, c["zipf"])
        if c["padding"] >= 0:
            ids[torch.rand(n, generator=g, device=DEV) < 0.5] = c["padding"]
        st.update(ids=ids, w=(rn(V, d) * 0.05).to(dt).requires_grad_(c["train"]))
        if c["train"]:
            st["gy"] = (rn(n, d) * 1e-3).to(dt)
    elif c["op"] == "balance":
        n, H, k, E = c["tokens"], c["heads"], c["top_k"], c["experts"]
        gates = torch.softmax(rn(n, H, k) * 1.5, -1).sort(-1, descending=True)[0]
        ids = _ids(g, (n, H, k), E, c["zipf"]).to(torch.int32)
        st.update(gates=gates.to(dt).requires_grad_(True), ids=ids)
    else:
        gs = [(rn(*s) * (1e-3 * (1.0 + i % 3))).to(dt) for i, s in enumerate(_clip_shapes(c))]
        size = sum(t.numel() for t in gs)
        # about the gradients' norm (or largest value), times `share`
        top = 1e-3 * (15.0 if c["norm"] == math.inf else 2.1 * math.sqrt(size)) * c["share"]
        # the clipped gradients go to one flat buffer, as the bucket of a reduction is
        flat = torch.empty(size, dtype=dt, device=DEV)
        st.update(grads=gs, flat=flat, out=[p.view_as(t) for p, t in zip(flat.split([t.numel() for t in gs]), gs)], max_norm=top)
    return st


# ---------------------------------------------------------------------------- the plain forms
def _ce_plain(h, w, labels, reduction, gy):
    hf, wf = h.detach().float(), w.detach().float()
    valid = labels != -100
    at = torch.where(valid, labels, torch.zeros_like(labels))[:, None]
    logits = hf @ wf.T
    top = logits.max(1, keepdim=True)[0]
    lse = (logits - top).exp().sum(1).log() + top[:, 0]
    rows = torch.where(valid, lse - logits.gather(1, at)[:, 0], torch.zeros_like(lse))
    count = valid.sum().float()
    loss = rows if reduction == "none" else rows.sum() if reduction == "sum" else rows.sum() / count
    if gy is None:
        return loss
    g = torch.where(valid, gy / count if reduction == "mean" else gy, torch.zeros_like(lse))
    p = (logits - lse[:, None]).exp_() * g[:, None]
    p.scatter_add_(1, at, -g[:, None])
    return loss, (p @ wf).to(h.dtype), (p.T @ hf).to(w.dtype)


def _embed_plain(ids, w, scale, padding, gy):
    y = (w.detach()[ids].float() * scale).to(w.dtype)
    if gy is None:
        return y
    g = gy.float()
    if padding >= 0:
        g = g * (ids != padding)[:, None]
    dw = torch.zeros(w.shape, device=w.device).index_add_(0, ids, g) * scale
    return y, dw.to(w.dtype)


def _balance_plain(gates, ids, experts):
    n, H, k = gates.shape
    e = ids.reshape(-1).long()
    counts = torch.zeros(experts, device=e.device, dtype=torch.int32).index_add_(0, e, torch.ones_like(e, dtype=torch.int32))
    f = counts.float() / (n * H * k)
    share = torch.zeros(experts, device=e.device).index_add_(0, e, gates.detach().float().reshape(-1)) / (n * H)
    loss = (f * share).sum() * experts
    return loss, counts, (f[e] * (experts / (n * H))).view_as(gates).to(gates.dtype)


def _clip_plain(grads, max_norm, norm, out):
    if norm == math.inf:
        total = torch.stack([t.float().abs().max() for t in grads]).max()
    else:
        total = torch.stack([(t.float() * t.float()).sum() for t in grads]).sum().sqrt()
    coef = (max_norm / (total + 1e-6)).clamp(max=1.0)
    for t, o in zip(grads, out):
        o.copy_(t.float() * coef)
    return total


def run(st):
    c = st["case"]
    if not own:
        if c["op"] == "ce":
            return _ce_plain(st["h"], st["w"], st["labels"], c["reduction"], st.get("gy"))
        if c["op"] == "embed":
            return _embed_plain(st["ids"], st["w"], c["scale"], c["padding"], st.get("gy"))
        if c["op"] == "balance":
            return _balance_plain(st["gates"], st["ids"], c["experts"])
        return _clip_plain(st["grads"], st["max_norm"], c["norm"], st["out"]), st["flat"]
    import ethos_amd

    if c["op"] == "ce":
        loss = ethos_amd.linear_cross_entropy(st["h"], st["w"], st["labels"], ignore_index=-100, reduction=c["reduction"])
        if not c["train"]:
            return loss
        return (loss.detach(), *torch.autograd.grad(loss, (st["h"], st["w"]), st["gy"]))
    if c["op"] == "embed":
        y = ethos_amd.embedding(st["ids"], st["w"], scale=c["scale"], padding_idx=c["padding"] if c["padding"] >= 0 else None)
        if not c["train"]:
            return y
        return y.detach(), torch.autograd.grad(y, st["w"], st["gy"])[0]
    if c["op"] == "balance":
        loss, counts = ethos_amd.balance_loss(st["gates"], st["ids"], c["experts"])
        return loss.detach(), counts, torch.autograd.grad(loss, st["gates"])[0]
    total = ethos_amd.clip_grads(st["grads"], st["max_norm"], norm_type=c["norm"], out=st["out"])
    return total, st["flat"]


# --------------------------------------------------------------------------------- the work
def work(c):
    b = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "ce":
        n, d, V = c["tokens"], c["d"], c["vocab"]
        io = (n * d + V * d) * b
        loss = 4 * n if c["reduction"] == "none" else 4
        labelled = max(1.0, n * (1.0 - c["ignored"]))
        return {"bytes": io * (2 if c["train"] else 1) + 8 * n + loss, "flops": (6.0 if c["train"] else 2.0) * labelled * V * d}
    if c["op"] == "embed":
        n, d, V = c["tokens"], c["d"], c["vocab"]
        fwd = 8 * n + (min(n, V) + n) * d * b
        return {"bytes": fwd + ((n + V) * d * b if c["train"] else 0), "flops": float(n * d * (2 if c["train"] else 1))}
    if c["op"] == "balance":
        p = c["tokens"] * c["heads"] * c["top_k"]
        return {"bytes": p * (4 + 2 * b) + 4 * c["experts"], "flops": 3.0 * p}
    size = sum(math.prod(s) for s in _clip_shapes(c))
    return {"bytes": 2 * b * size, "flops": 3.0 * size}


# ------------------------------------------------------------------------------- in float64
def exact(case, seed):
    st, c = prepare(case, seed), case
    f = torch.float64
    with torch.no_grad():
        if c["op"] == "ce":
            h, w, labels = st["h"].detach().to(f), st["w"].detach().to(f), st["labels"]
            keep = torch.nonzero(labels >= 0)[:, 0]
            loss = torch.zeros(len(labels), dtype=f, device=DEV)
            dh, dw = torch.zeros_like(h), torch.zeros_like(w)
            gy = st.get("gy")
            for part in keep.split(1024):
                x = h[part]
                logp = torch.log_softmax(x @ w.t(), dim=1)
                loss[part] = -logp[torch.arange(len(part), device=DEV), labels[part]]
                if c["train"]:
                    err = logp.exp_()
                    err[torch.arange(len(part), device=DEV), labels[part]] -= 1.0
                    err *= (gy[part].to(f) if c["reduction"] == "none" else gy.to(f) / (len(keep) if c["reduction"] == "mean" else 1)).reshape(-1, 1)
                    dh[part] = err @ w
                    dw += err.t() @ x
            if c["reduction"] != "none":
                loss = loss.sum() / (len(keep) if c["reduction"] == "mean" else 1)
            return (loss, dh, dw) if c["train"] else loss
        if c["op"] == "embed":
            w, ids = st["w"].detach().to(f), st["ids"]
            y = torch.index_select(w, 0, ids).mul_(c["scale"])
            if not c["train"]:
                return y
            order = torch.argsort(ids)
            if c["padding"] >= 0:
                order = order[ids[order] != c["padding"]]
            dw = torch.zeros_like(w)
            dw.index_put_((ids[order],), st["gy"].to(f)[order] * c["scale"], accumulate=True)
            return y, dw
        if c["op"] == "balance":
            gates, e = st["gates"].detach().to(f), st["ids"].long()
            n, H, k = gates.shape
            counts = torch.bincount(e.flatten(), minlength=c["experts"])
            slope = counts.to(f)[e] * (c["experts"] / (float(n) * H * k) / (float(n) * H))
            return (slope * gates).sum(), counts.to(torch.int32), slope
        if c["norm"] == math.inf:
            total = max(t.abs().max().to(f) for t in st["grads"])
        else:
            total = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(t.to(f)) for t in st["grads"]]))
        scale = torch.minimum(torch.ones_like(total), st["max_norm"] / (total + 1e-6))
        return total, torch.cat([t.flatten().to(f) * scale for t in st["grads"]])
