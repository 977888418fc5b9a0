"""Operators of serving the language model from a cache: what is timed and compared.

`listed()` names the cases, `draw(rng)` gives further ones of the same ranges, `prepare` makes
what a program holds before the call, `run` makes one pass (in plain torch operations, or with
`own` through this package), `exact` is the same function in float64.  Four operators:

  append  latent_append: the new tokens' rows of a cache of latents in pages: each row's latent
          normalised, its rotary key rotated by the token's position
  attend  paged_attention: attention of the new tokens of several sequences over that cache
  copy    copy_pages: pages of the cache of every block copied, for a fork or a compaction
  verify  verify_drafts: drafted tokens accepted or not by the model's probabilities from given
          random numbers, and the token that follows them

A cache is [pages, page tokens, latent width + rotary width]; a sequence is a row of a table of
page numbers and a length; the batch's new tokens are rows, those of sequence i from starts[i]
to starts[i + 1], and the last ones of its length.  All inputs are made on the GPU from the seed."""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
VOCAB = 100277  # the language model's vocabulary
BASE = 10000.0  # of its rotary rates
EPS = 1e-6      # of its norms


def _attend(seqs, new, length, **kw):
    """`seqs` sequences of up to `new` new tokens and up to `length` tokens in all."""
    return dict(dict(op="attend", seqs=seqs, new=new, length=length, ragged=True, heads=16, rank=256, rope=64, nope=64, v=64, page=64,
                     dtype="bf16"), **kw)


def _append(seqs, new, length, **kw):
    return dict(dict(op="append", seqs=seqs, new=new, length=length, ragged=True, q_rank=768, rank=256, rope=64, page=64, dtype="bf16"), **kw)


def _copy(blocks, pages, pairs, **kw):
    return dict(dict(op="copy", blocks=blocks, pages=pages, pairs=pairs, page=64, width=320, dtype="bf16"), **kw)


def _verify(seqs, drafts, **kw):
    return dict(dict(op="verify", seqs=seqs, drafts=drafts, vocab=VOCAB, dtype="bf16", probs="fp32", ragged=True, temperature=1.0), **kw)


def listed():
    return [
        # a decode step of 64 conversations of up to 8,192 tokens
        dict(_attend(64, 1, 8192), name="attend_decode_64"),
        # a decode step of one conversation over a long document
        dict(_attend(1, 1, 65536, ragged=False), name="attend_decode_1_long"),
        # the step that checks four drafted tokens of 16 conversations
        dict(_attend(16, 5, 4096), name="attend_drafts_16"),
        # a chunk of 2,048 tokens of a long prompt, in pages of another size
        dict(_attend(1, 2048, 7001, ragged=False, page=128), name="attend_chunk_2048"),
        # short prompts and follow-ups of a small float32 model, odd sizes
        dict(_attend(5, 33, 300, heads=4, rank=32, rope=16, nope=16, v=16, page=16, dtype="fp32"), name="attend_fp32_5"),
        # the rows of a decode step's tokens
        dict(_append(64, 1, 8192), name="append_decode_64"),
        # the rows of a batch of prompts, far into long texts
        dict(_append(4, 2048, 100000, ragged=False), name="append_prompt_8192"),
        # the pages that 64 forked sequences begin to write in, of a model of 12 blocks
        dict(_copy(12, 256, 64), name="copy_fork_64"),
        # a cache moved together, one page in three
        dict(_copy(6, 900, 300), name="copy_compact_300"),
        # four drafted tokens of each of 64 sequences, sampled from a draft model's probabilities
        dict(_verify(64, 4), name="verify_64x4"),
        # no drafts: one token sampled for one sequence
        dict(_verify(1, 0, temperature=0.8), name="verify_1x0"),
        # eight tokens drafted without probabilities (looked up in the text), float32 logits, an odd vocabulary
        dict(_verify(16, 8, vocab=8009, dtype="fp32", probs="none"), name="verify_fp32_16x8"),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "drafts", "chunk", "attend_fp32", "append", "copy", "verify", "verify"])
    if op == "decode":
        seqs = _log(rng, 1, 64)
        return _attend(seqs, 1, _log(rng, 60, min(65536, 524288 // seqs)), heads=rng.choice([4, 8, 12, 16, 16, 32]),
                       page=rng.choice([16, 64, 128]))
    if op == "drafts":
        seqs = _log(rng, 1, 32)
        return _attend(seqs, rng.randint(2, 12), _log(rng, 60, min(32768, 131072 // seqs)), heads=rng.choice([8, 16, 16]),
                       page=rng.choice([16, 64, 128]))
    if op == "chunk":
        new = _log(rng, 40, 2048)
        return _attend(rng.randint(1, max(1, min(8, 2048 // new))), new, new + _log(rng, 1, 4000), heads=rng.choice([8, 16, 16]),
                       page=rng.choice([16, 64, 128, 256]))
    if op == "attend_fp32":
        rank = rng.choice([32, 64, 128])
        return _attend(_log(rng, 1, 8), _log(rng, 1, 64), _log(rng, 70, 600), heads=rng.choice([2, 4, 8]), rank=rank, rope=rng.choice([16, 32]),
                       nope=rng.choice([16, 32]), v=rng.choice([16, 32, 48]), page=rng.choice([8, 16, 64]), dtype="fp32")
    if op == "append":
        big = rng.random() < 0.5
        return _append(_log(rng, 1, 8), _log(rng, 1, 1024) if big else 1, _log(rng, 1100, 100000), rank=rng.choice([128, 256, 256, 512]),
                       page=rng.choice([16, 64, 128]), dtype=rng.choice(["bf16", "bf16", "fp32"]))
    if op == "copy":
        pages = _log(rng, 16, 900)
        return _copy(rng.randint(1, 6), pages, _log(rng, 1, pages // 2), page=rng.choice([16, 64]), dtype=rng.choice(["bf16", "bf16", "fp32"]))
    return _verify(_log(rng, 1, 64), rng.choice([0, 1, 2, 3, 4, 4]), vocab=_log(rng, 500, VOCAB), dtype=rng.choice(["bf16", "bf16", "fp32"]),
                   probs=rng.choice(["fp32", "fp32", "bf16", "none"]), temperature=rng.choice([1.0, 1.0, 0.7, 1.3, 0.0]))


# ------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _plan(c):
    """(total lengths, new tokens) of each sequence: the first has all, others less where ragged.
    The same for every seed, as the work is."""
    i = torch.arange(c["seqs"], dtype=torch.float64)
    frac = (i * 0.6180339887498949) % 1.0 if c["ragged"] else torch.zeros_like(i)
    new = (c["new"] - frac * 0.5 * c["new"]).ceil().long().clamp(min=1)
    length = (c["length"] * (1.0 - 0.9 * frac)).ceil().long()
    return torch.maximum(length, new).tolist(), new.tolist()


def _batch(c, g):
    """The batch on the device: a table of scattered pages, lengths, where each sequence's rows begin, and the
    number of pages of the cache."""
    lens, new = _plan(c)
    each = [-(-n // c["page"]) for n in lens]
    total = sum(each) + 3
    numbers = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.full((c["seqs"], max(each) + 1), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, k in enumerate(each):
        table[i, :k] = numbers[at:at + k]
        at += k
    starts = [0]
    for k in new:
        starts.append(starts[-1] + k)
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"table": table, "lens": dev(lens), "starts": dev(starts), "host_lens": lens, "host_new": new}, total


def _rates(rope):
    return 1.0 / BASE ** (torch.arange(0, rope, 2, device=DEV, dtype=torch.float32) / rope)


def prepare(case, seed):
    g = _gen(seed)
    c, dt = case, DTYPES[case["dtype"]]
    st = {"case": case}
    rn = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    if c["op"] == "attend":
        batch, pages = _batch(c, g)
        n, H = sum(batch["host_new"]), c["heads"]
        # the cache as latent_append leaves it; memory that no token has filled holds NaN
        pool = torch.full((pages, c["page"], c["rank"] + c["rope"]), math.nan, dtype=dt, device=DEV)
        for i, length in enumerate(batch["host_lens"]):
            p = torch.arange(length, device=DEV)
            pool[batch["table"][i].long()[p // c["page"]], p % c["page"]] = rn(length, c["rank"] + c["rope"]).to(dt)
        w = (rn(H * (c["nope"] + c["v"]), c["rank"]) / math.sqrt(c["rank"])).to(dt)
        q = (rn(n, H, c["nope"] + c["rope"]) * 1.5).to(dt)
        st.update(batch, q=q, w=w, pool=pool, rates=_rates(c["rope"]), scale=1.0 / math.sqrt(c["nope"] + c["rope"]))
    elif c["op"] == "append":
        batch, pages = _batch(c, g)
        n = sum(batch["host_new"])
        # the projection's output: the query's latent, the latent, the rotary key
        a = (rn(n, c["q_rank"] + c["rank"] + c["rope"]) * (0.2 + rn(n, 1).abs())).to(dt)
        pool = torch.zeros(pages, c["page"], c["rank"] + c["rope"], dtype=dt, device=DEV)
        st.update(batch, rows=a[:, c["q_rank"]:], gain=(1.0 + 0.1 * rn(c["rank"])).to(dt), pool=pool, rates=_rates(c["rope"]))
    elif c["op"] == "copy":
        pool = rn(c["blocks"], c["pages"], c["page"], c["width"]).to(dt)
        at = torch.randperm(c["pages"], generator=g, device=DEV).tolist()
        st.update(pool=pool, src=at[:c["pairs"]], dst=at[c["pairs"]:2 * c["pairs"]])
    else:
        b, m, V = c["seqs"], c["drafts"], c["vocab"]
        # peaked distributions, the draft model's near the target's
        logits = (rn(b, m + 1, V) * 2.5).to(dt)
        noisy = logits[:, :m].float() + rn(b, m, V) * 0.7
        p = torch.softmax(noisy, -1)
        drafts = torch.multinomial(p.view(-1, V), 1, generator=g).view(b, m) if b * m else torch.zeros(b, m, dtype=torch.int64, device=DEV)
        if c["probs"] == "none":
            drafts = noisy.argmax(-1)
        counts = torch.tensor([m - (i * 7) % (m + 1) // 2 if c["ragged"] else m for i in range(b)], dtype=torch.int32, device=DEV)
        st.update(logits=logits, drafts=drafts, counts=counts, probs=None if c["probs"] == "none" else p.to(DTYPES[c["probs"]]),
                  u_accept=torch.rand(b, m, generator=g, device=DEV), u_sample=torch.rand(b, generator=g, device=DEV))
    return st


# ---------------------------------------------------------------------------- the plain forms
def _rotated(r, positions, rates):
    """[a, b] -> [a cos - b sin, b cos + a sin] in 32 bits, the angles in 64."""
    t = positions.double()[:, None] * rates.double()
    c, s = t.cos().float(), t.sin().float()
    shape = (len(positions),) + (1,) * (r.dim() - 2) + (-1,)
    c, s = c.view(shape), s.view(shape)
    a, b = r.float().chunk(2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def _attend_plain(st):
    c, out = st["case"], []
    H, R, nope = c["heads"], c["rank"], c["nope"]
    w = st["w"].float().view(H, nope + c["v"], R)
    at = 0
    for i, (length, new) in enumerate(zip(st["host_lens"], st["host_new"])):
        p = torch.arange(length, device=DEV)
        rows = st["pool"][st["table"][i].long()[p // c["page"]], p % c["page"]].float()
        k = (rows[:, :R] @ w[:, :nope].reshape(-1, R).T).view(length, H, nope).transpose(0, 1).contiguous()
        v = (rows[:, :R] @ w[:, nope:].reshape(-1, R).T).view(length, H, c["v"]).transpose(0, 1).contiguous()
        q = st["q"][at:at + new].float()
        turned = _rotated(q[..., nope:], p[length - new:], st["rates"]).transpose(0, 1)
        s = q[..., :nope].transpose(0, 1) @ k.transpose(1, 2) + turned @ rows[:, R:].T
        s = s * st["scale"]
        s.masked_fill_(p[None, None, :] > p[length - new:][None, :, None], -math.inf)
        e = (s - s.amax(-1, keepdim=True)).exp_()
        o = (e @ v) / e.sum(-1, keepdim=True)
        out.append(o.transpose(0, 1).reshape(new, H * c["v"]))
        at += new
    return torch.cat(out).to(st["q"].dtype)


def _append_plain(st):
    c = st["case"]
    new = torch.tensor(st["host_new"], device=DEV)
    which = torch.repeat_interleave(torch.arange(len(new), device=DEV), new)
    pos = torch.arange(len(which), device=DEV) - st["starts"].long()[which] + st["lens"].long()[which] - new[which]
    x = st["rows"][:, :c["rank"]].float()
    y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * st["gain"].float()
    k = _rotated(st["rows"][:, c["rank"]:], pos, st["rates"])
    st["pool"][st["table"].long()[which, pos // c["page"]], pos % c["page"]] = torch.cat((y, k), -1).to(st["pool"].dtype)
    return st["pool"]


def _copy_plain(st):
    st["pool"][:, st["dst"]] = st["pool"][:, st["src"]]
    return st["pool"]


def _verify_plain(st):
    """In 64 bits: whether a random number lies below a sum must not hang on its rounding."""
    c, logits = st["case"], st["logits"].double()
    b, m, V = c["seqs"], c["drafts"], c["vocab"]
    if c["temperature"] == 0.0:
        p = torch.zeros_like(logits).scatter_(2, logits.argmax(-1, keepdim=True), 1.0)
    else:
        e = ((logits - logits.amax(-1, keepdim=True)) / c["temperature"]).exp_()
        p = e / e.sum(-1, keepdim=True)
    at = st["drafts"][:, :, None]
    q = torch.zeros(b, m, V, dtype=torch.float64, device=DEV).scatter_(2, at, 1.0) if st["probs"] is None else st["probs"].double()
    ok = st["u_accept"].double() * q.gather(2, at)[..., 0] < p[:, :m].gather(2, at)[..., 0]
    ok &= torch.arange(m, device=DEV) < st["counts"][:, None]
    accepted = ok.long().cumprod(1).sum(1)
    row = torch.arange(b, device=DEV)
    left = p[row, accepted]
    if m:
        after = (accepted < st["counts"]).double()[:, None]
        left = (left - q[row, accepted.clamp(max=m - 1)] * after).clamp_(min=0.0)
    sums = left.cumsum(1)
    token = torch.searchsorted(sums, st["u_sample"].double()[:, None] * sums[:, -1:], right=True)[:, 0]
    return accepted.int(), token


def run(st):
    op = st["case"]["op"]
    if not own:
        return {"attend": _attend_plain, "append": _append_plain, "copy": _copy_plain, "verify": _verify_plain}[op](st)
    import ethos_amd

    if op == "attend":
        return ethos_amd.paged_attention(st["q"], st["w"], st["pool"], st["table"], st["lens"], st["starts"], st["rates"], st["scale"])
    if op == "append":
        ethos_amd.latent_append(st["rows"], st["gain"], st["pool"], st["table"], st["lens"], st["starts"], st["rates"], eps=EPS)
        return st["pool"]
    if op == "copy":
        ethos_amd.copy_pages(st["pool"], st["src"], st["dst"])
        return st["pool"]
    return ethos_amd.verify_drafts(st["logits"], st["drafts"], st["u_accept"], st["u_sample"], draft_probs=st["probs"], counts=st["counts"],
                                   temperature=st["case"]["temperature"])


# --------------------------------------------------------------------------------- the work
def work(c):
    b = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "attend":
        lens, new = _plan(c)
        H, R, P, D, v = c["heads"], c["rank"], c["rope"], c["nope"], c["v"]
        flops = 0.0
        for length, m in zip(lens, new):
            pairs = m * (length - (m - 1) / 2) * H
            # the products with the weight go to the keys and values, or to the queries and outputs
            keys = 2.0 * length * H * (D + v) * R + 2.0 * pairs * (D + P + v)
            queries = 2.0 * m * H * (D + v) * R + 2.0 * pairs * (2 * R + P)
            flops += min(keys, queries)
        n = sum(new)
        return {"bytes": (sum(lens) * (R + P) + n * H * (D + P + v) + H * (D + v) * R) * b, "flops": flops}
    if c["op"] == "append":
        n = sum(_plan(c)[1])
        return {"bytes": 2 * n * (c["rank"] + c["rope"]) * b, "flops": n * (4.0 * c["rank"] + 3.0 * c["rope"])}
    if c["op"] == "copy":
        return {"bytes": 2 * c["blocks"] * c["pairs"] * c["page"] * c["width"] * b, "flops": 0.0}
    rows, V = c["seqs"] * (c["drafts"] + 1), c["vocab"]
    q = 0 if c["probs"] == "none" or c["drafts"] == 0 else 2 if c["probs"] == "bf16" else 4
    # of the drafts' probabilities one row of a sequence
    return {"bytes": rows * V * b + c["seqs"] * V * q, "flops": 3.0 * rows * V}


# ------------------------------------------------------------------------------- in float64
def exact(case, seed):
    st, c, f = prepare(case, seed), case, torch.float64
    with torch.no_grad():
        if c["op"] == "attend":
            # the weight goes to the queries and to the weighted sums of latents
            H, R, D = c["heads"], c["rank"], c["nope"]
            w = st["w"].to(f).reshape(H, D + c["v"], R)
            flat = st["pool"].to(f).reshape(-1, R + c["rope"])
            out = torch.empty(len(st["q"]), H, c["v"], dtype=f, device=DEV)
            starts = st["starts"].tolist()
            for i, length in enumerate(st["lens"].tolist()):
                slot = torch.cat([torch.arange(int(t) * c["page"], (int(t) + 1) * c["page"], device=DEV)
                                  for t in st["table"][i].tolist() if t >= 0])[:length]
                rows = flat[slot]
                q = st["q"][starts[i]:starts[i + 1]].to(f)
                first = length - len(q)
                turn = torch.polar(torch.ones((), dtype=f, device=DEV),
                                   torch.arange(first, length, device=DEV, dtype=f)[:, None] * st["rates"].to(f)[None, :])
                half = c["rope"] // 2
                seen = torch.ones(len(q), length, dtype=torch.bool, device=DEV).tril(first)
                for h in range(H):
                    z = torch.complex(q[:, h, D:D + half], q[:, h, D + half:]) * turn
                    big = torch.cat((q[:, h, :D] @ w[h, :D], z.real, z.imag), 1)
                    logit = torch.where(seen, (big @ rows.t()) * st["scale"], -math.inf)
                    out[starts[i]:starts[i + 1], h] = torch.softmax(logit, 1) @ rows[:, :R] @ w[h, D:].t()
            return out.reshape(len(out), -1)
        if c["op"] == "append":
            pool = st["pool"].to(f)
            x = st["rows"].to(f)
            starts, half = st["starts"].tolist(), c["rope"] // 2
            for i, length in enumerate(st["lens"].tolist()):
                mine = x[starts[i]:starts[i + 1]]
                pos = torch.arange(length - len(mine), length, device=DEV)
                lat = mine[:, :c["rank"]]
                lat = lat * torch.rsqrt(lat.pow(2).sum(1, keepdim=True) / c["rank"] + EPS) * st["gain"].to(f)
                z = torch.complex(mine[:, c["rank"]:c["rank"] + half], mine[:, c["rank"] + half:])
                z = z * torch.exp(1j * pos.to(f)[:, None] * st["rates"].to(f))
                slot = st["table"][i].long().index_select(0, pos.div(c["page"], rounding_mode="floor")) * c["page"] + pos.remainder(c["page"])
                pool.view(-1, pool.shape[-1])[slot] = torch.cat((lat, z.real, z.imag), 1)
            return pool
        if c["op"] == "copy":
            pool = st["pool"].to(f)
            for s, d in zip(st["src"], st["dst"]):
                pool[:, d].copy_(pool[:, s])
            return pool
        accepted, tokens = [], []
        for i in range(c["seqs"]):
            n = int(st["counts"][i])
            z = st["logits"][i].to(f)
            p = torch.softmax(z / c["temperature"], -1) if c["temperature"] > 0 else torch.nn.functional.one_hot(z.argmax(-1), c["vocab"]).to(f)
            a, rest = 0, None
            for j in range(n):
                x = int(st["drafts"][i, j])
                q = torch.nn.functional.one_hot(st["drafts"][i, j], c["vocab"]).to(f) if st["probs"] is None else st["probs"][i, j].to(f)
                if float(st["u_accept"][i, j]) * float(q[x]) < float(p[j, x]):
                    a += 1
                    continue
                rest = (p[j] - q).clamp(min=0.0)
                break
            rest = p[n] if rest is None else rest
            run_sum = torch.cumsum(rest, 0)
            accepted.append(a)
            tokens.append(int((run_sum <= float(st["u_sample"][i]) * run_sum[-1]).sum()))
        return torch.tensor(accepted, dtype=torch.int32, device=DEV), torch.tensor(tokens, device=DEV)
