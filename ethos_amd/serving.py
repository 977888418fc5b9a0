"""Operators of serving the language model from a cache, as HIP kernels (include/ethos_hip.h):

  latent_append    the new tokens' rows of a cache of latents: normalised latent, rotated key
  paged_attention  latent attention of the new tokens over the cache
  copy_pages       pages of the cache copied, in every block's part at once
  verify_drafts    drafted tokens accepted or not by the model's probabilities, the token after them
  LatentCache      the pages of a cache, and which sequence has which: extend, truncate, fork, free, compact

CompressedMoEModel.extend and .speculate run them in the model's blocks.

The reference has no cache and decodes nothing; its attention forms every token's keys and values anew
(model.py:104-160).  Inputs are HIP tensors on the current device, bf16 or float32; there is no CPU path.
All work goes to the current stream.  Results are the same on every run.  The operators have no gradients:
tensors that ask for one, forward-mode derivatives and torch.jit.trace are refused."""
from __future__ import annotations

import operator
from array import array
from typing import NamedTuple

import torch

from . import hip, training

__all__ = ["Batch", "LatentCache", "copy_pages", "latent_append", "paged_attention", "verify_drafts"]


_requires_grad = operator.attrgetter("requires_grad")


def _check(what: str, *ts) -> None:
    """Refuses what the kernels would hide from autograd, and other devices than the current one."""
    if training._is_followed():
        training._refuse_followed(what, *ts)
    try:
        devices = set(map(torch.Tensor.get_device, ts))
    except TypeError:
        devices = {-1}
    if -1 in devices or devices != {hip._current_device()}:
        for t in ts:
            training._device_check(f"{what}: an input", t)
    if torch.is_grad_enabled() and any(map(_requires_grad, ts)):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")


def _written(t: torch.Tensor) -> None:
    """t was written by address."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [n, d], or a copy of it, as rows that the kernels can read: evenly spaced, 16-byte aligned."""
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and (t.stride(0) * t.element_size() % 16 == 0 and t.stride(0) >= t.shape[1] or t.shape[0] < 2):
        return t
    return training._dense(t)


def latent_append(rows: torch.Tensor, gain: torch.Tensor, pool: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                  starts: torch.Tensor, rates: torch.Tensor, eps: float = 1e-6) -> None:
    """Writes the new tokens of a batch into a cache of latents.

    rows [n, rank + rope]: each token's latent and rotary key as they leave the projection (rows evenly spaced, for
    example a part of a wider one); gain [rank]: the latent's RMSNorm; pool [pages, page, rank + rope], contiguous, the
    page a power of two.  Sequence i has the pages table[i] (int32 [sequences, width]) and lens[i] tokens (int32), the new
    ones included, which are rows starts[i] .. starts[i + 1] - 1 (int32 [sequences + 1], ascending).  Their place in the cache
    gets the normalised latent (gain x / sqrt(mean(x^2) + eps)) and the key rotated by position times rates
    (float32 [rope / 2], Rotary.rates), computed in float32 and rounded once.  Rows of no sequence, positions
    without a page and pages outside the pool are left out.  The sequences' new tokens may not share places."""
    _check("latent_append", rows, gain, pool, table, lens, starts, rates)
    if pool.dim() != 3 or rows.dim() != 2 or gain.dim() != 1 or rows.shape[1] != pool.shape[2] or gain.shape[0] > pool.shape[2]:
        raise RuntimeError(f"latent_append: inconsistent shapes {tuple(rows.shape)}, {tuple(gain.shape)} and {tuple(pool.shape)}")
    if pool.dtype not in hip.FLOATS or rows.dtype != pool.dtype or gain.dtype != pool.dtype:
        raise TypeError(f"rows, gain and pool must all be bfloat16 or all float32, got {rows.dtype}, {gain.dtype} and {pool.dtype}")
    hip.latent_append(_rows(rows), training._dense(gain), pool, table, lens, starts, rates, eps)
    _written(pool)


def paged_attention(q: torch.Tensor, weight: torch.Tensor, pool: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                    starts: torch.Tensor, rates: torch.Tensor, scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """Latent attention of a batch's new tokens over the cache that latent_append filled: [n, heads v_dim].

    q [n, heads, nope + rope], the rotary part not yet rotated; weight [heads (nope + v_dim), rank], kv_b_proj's;
    pool, table, lens, starts and rates as latent_append takes them.  A token sees its sequence's positions up to its own:
    softmax(scale q k) v over them (scale positive, at most 1e35), with k = [weight's nope rows of the head times the latent | the
    cached key] and v its v_dim rows times the latent.  One token a sequence, a few or thousands: any mixture, though a batch
    takes one form, and long chunks beside single tokens are faster in two calls.  Rows of no sequence are left as they are
    (`out`, or uninitialised); a token that sees nothing has zeros; one that sees a position without a page, a latent that is not
    finite or a key that is NaN, NaN.  An infinite key gives NaN, or no weight where the score is -inf; if all are, NaN.

    Scores and sums are float32; in bf16 (rank 256, rope 64, pages of 8 tokens or more) products take bf16 operands, and where
    sequences have 96 new tokens or more on the average, and nope and v_dim are 64, fp16 ones: there a query or a key of 2^20 and
    more, or a value of 2^18, counts as infinite, and steps are no finer than 2^-20 of a query or key and 2^-22 of a value, fewer
    bits than bf16's below 2^-13 and 2^-15.  `out`: a contiguous tensor for the result, apart from the inputs."""
    _check("paged_attention", q, weight, pool, table, lens, starts, rates, *(() if out is None else (out,)))
    if q.dim() != 3 or weight.dim() != 2 or pool.dim() != 3:
        raise RuntimeError(f"paged_attention: q, weight and pool must have 3, 2 and 3 dims, got {tuple(q.shape)}, {tuple(weight.shape)} and "
                           f"{tuple(pool.shape)}")
    o = hip.paged_attention(training._dense(q), training._dense(weight), pool, table, lens, starts, rates, scale, out)
    if out is not None:
        _written(out)
    return o


def _page_list(name: str, v) -> array:
    if isinstance(v, torch.Tensor):
        if v.is_cuda:
            raise TypeError(f"copy_pages: {name} must be on the host (a list, or a CPU tensor)")
        v = v.tolist()
    return array("i", v if isinstance(v, list) else list(v))


def _page_pairs(src, dst) -> tuple[array, array]:
    """Which pages are copied where, checked (as plain numbers: tensors of one value would be told apart by what they are)."""
    src, dst = _page_list("src", src), _page_list("dst", dst)
    if len(src) != len(dst):
        raise ValueError(f"copy_pages: {len(src)} pages to copy but {len(dst)} places")
    to = set(dst)
    if len(to) != len(dst) or not to.isdisjoint(src):
        raise ValueError("copy_pages: a page is written twice, or both read and written")
    return src, dst


def copy_pages(pool: torch.Tensor, src, dst) -> None:
    """Copies page src[i] to page dst[i], for every i, in all blocks (65,535 at most) of pool [blocks, pages, ...] (contiguous,
    any dtype of two or four bytes).  src and dst: sequences of whole numbers on the host, read during the call; no page may be written
    twice or both read and written."""
    _check("copy_pages", pool)
    if pool.dim() < 3 or not pool.is_contiguous() or pool.element_size() not in (2, 4):
        raise RuntimeError(f"copy_pages: pool must be contiguous [blocks, pages, ...] of 2 or 4 bytes a value, got {tuple(pool.shape)} "
                           f"{pool.dtype}")
    hip.copy_pages(pool, *_page_pairs(src, dst))
    _written(pool)


def verify_drafts(logits: torch.Tensor, drafts: torch.Tensor, u_accept: torch.Tensor, u_sample: torch.Tensor,
                  draft_probs: torch.Tensor | None = None, counts: torch.Tensor | None = None, temperature: float = 1.0):
    """(accepted int32 [b], tokens int64 [b]): how many drafted tokens of each sequence stand, and the token after them.

    logits [b, m + 1, vocab] (bf16 or float32): row j follows draft j - 1, row 0 the last token before the drafts;
    drafts int64 [b, m], of which a sequence has counts[i] (int32 [b]; all m without it); draft_probs [b, m, vocab]
    (bf16 or float32): what each was drawn from, None where it had probability 1; u_accept [b, m] and u_sample [b]: float32,
    uniform in [0, 1).  With p_j = softmax(logits_j / temperature) (0: 1 at the first largest logit), draft j stands if all
    before it do and u_accept q_j(x_j) < p_j(x_j).  The token is drawn from max(p_a - q_a, 0) behind the a-th (from p_a if all
    stand, or that is 0 everywhere): the lowest index whose weights up to it exceed u_sample of their sum.  Tokens and drafts
    together are then distributed as p's.  Without drafts (m = 0) it samples.  Words may be masked by logits of -inf.  A
    token is -1 where its row of logits has a NaN, no finite one, or one that is +inf (with a temperature), and where the row of
    draft_probs that is subtracted (with a temperature) has a NaN.  All in float64."""
    _check("verify_drafts", *[t for t in (logits, drafts, u_accept, u_sample, draft_probs, counts) if t is not None])
    if (logits.dtype not in hip.FLOATS or drafts.dtype != torch.int64 or u_accept.dtype != torch.float32 or u_sample.dtype != torch.float32
            or draft_probs is not None and draft_probs.dtype not in hip.FLOATS or counts is not None and counts.dtype != torch.int32):
        raise TypeError(f"verify_drafts takes logits and draft_probs of {' or '.join(map(str, hip.FLOATS))}, int64 drafts, float32 u_accept and "
                        f"u_sample and int32 counts, got {[t if t is None else t.dtype for t in (logits, draft_probs, drafts, u_accept, u_sample, counts)]}")
    dense = [None if t is None else t.contiguous() for t in (logits, drafts, draft_probs, counts, u_accept, u_sample)]
    return hip.verify(*dense, temperature)


# -------------------------------------------------------------------------- the cache
class Batch(NamedTuple):
    """New tokens of several sequences, as latent_append and paged_attention take them (int32, on the device)."""

    table: torch.Tensor   # [sequences, pages]
    lens: torch.Tensor    # [sequences], the new tokens included
    starts: torch.Tensor  # [sequences + 1]: the rows of each one's new tokens
    counts: list          # how many each has, on the host


class _Sequence:
    __slots__ = ("length", "pages")

    def __init__(self, length: int, pages: array):
        self.length, self.pages = length, pages


class LatentCache:
    """A cache of latents for `blocks` attention blocks in `pages` pages of `page` tokens (a power of two), and the
    sequences in it.  pool [blocks, pages, page, rank + rope] holds, per token and block, the normalised latent and the rotated
    key: in bf16 640 bytes for rank 256 and rope 64.  A page number stands for the same page of every block.

    Which page is whose is known on the host: no call waits for the device.  `extend` makes room for new tokens and
    gives the batch that the operators take; a fork shares its pages, and a shared page is copied when one of its
    sequences first writes in it.  The device's work (page copies, the batch's tensors) is enqueued on the current stream:
    use a cache on one stream, or let streams wait for each other.  `extend` and `compact` refuse to be captured into a graph,
    whose replays would read the batch from host memory long used again, and move pages that the books have moved already."""

    def __init__(self, blocks: int, rank: int, rope: int, pages: int, page: int = 64, dtype: torch.dtype = torch.bfloat16, device=None):
        if blocks <= 0 or pages <= 0 or rank <= 0 or rope < 0:
            raise ValueError(f"LatentCache: blocks, pages and rank must be positive, got {blocks}, {pages} and {rank}")
        if page <= 0 or page & (page - 1) or page > 65536:
            raise ValueError(f"LatentCache: page must be a power of two up to 65536, got {page}")
        if dtype not in hip.FLOATS:
            raise TypeError(f"LatentCache: dtype must be bfloat16 or float32, got {dtype}")
        self.page, self.rank, self.rope = page, rank, rope
        # (never-written memory is never read, but a NaN in it would be by a caller's own sums over pages)
        self.pool = torch.zeros((blocks, pages, page, rank + rope), dtype=dtype, device="cuda" if device is None else device)
        self._users = [0] * pages                       # sequences that have the page
        self._free = array("i", range(pages - 1, -1, -1))  # the lowest is given out first
        self._sequences: dict[int, _Sequence] = {}
        self._next = 0

    def _refuse_capture(self, what: str) -> None:
        if self.pool.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"LatentCache.{what} cannot be captured into a graph")

    @property
    def pages_free(self) -> int:
        return len(self._free)

    def _of(self, seq: int) -> _Sequence:
        try:
            return self._sequences[seq]
        except KeyError:
            raise KeyError(f"the cache has no sequence {seq}") from None

    def new(self) -> int:
        """An empty sequence's number."""
        seq, self._next = self._next, self._next + 1
        self._sequences[seq] = _Sequence(0, array("i"))
        return seq

    def length(self, seq: int) -> int:
        return self._of(seq).length

    def pages(self, seq: int) -> list:
        """The page numbers of a sequence, in order."""
        return self._of(seq).pages.tolist()

    def fork(self, seq: int) -> int:
        """A new sequence of the same tokens, on the same pages."""
        s = self._of(seq)
        new = self.new()
        self._sequences[new] = _Sequence(s.length, array("i", s.pages))
        for p in s.pages:
            self._users[p] += 1
        return new

    def _drop(self, pages) -> None:
        for p in pages:
            self._users[p] -= 1
            if self._users[p] == 0:
                self._free.append(p)

    def truncate(self, seq: int, length: int) -> None:
        """Forgets a sequence's tokens from `length` on."""
        s, length = self._of(seq), operator.index(length)
        if not 0 <= length <= s.length:
            raise ValueError(f"sequence {seq} has {s.length} tokens, it cannot be cut to {length}")
        self._cut(s, length)

    def _cut(self, s: _Sequence, length: int) -> None:
        keep = -(-length // self.page)
        self._drop(reversed(s.pages[keep:]))
        del s.pages[keep:]
        s.length = length

    def free(self, seq: int) -> None:
        """Forgets a sequence."""
        self.truncate(seq, 0)
        del self._sequences[seq]

    def extend(self, seqs, counts) -> Batch:
        """Room for counts[i] new tokens of sequence seqs[i]: their batch, in that order.  With too few free pages it raises
        RuntimeError and changes nothing."""
        self._refuse_capture("extend")
        seqs, counts = list(seqs), [operator.index(c) for c in counts]
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(c < 0 for c in counts):
            raise ValueError("extend: each sequence once, with the number of its new tokens")
        own = [self._of(q) for q in seqs]
        # shared pages that new tokens go to; of several batch sequences that share one, each but a last sole user copies it
        copies, users = [], {}
        need = 0
        for i, (s, c) in enumerate(zip(own, counts)):
            need += -(-(s.length + c) // self.page) - len(s.pages)
            if c and s.length % self.page:
                p = s.pages[-1]
                left = users.get(p, self._users[p])
                if left > 1:
                    copies.append(i)
                    users[p] = left - 1
        if need + len(copies) > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, {need + len(copies)} are needed")
        if copies:  # (the books behind the copies: a refused copy changes nothing)
            src, dst = [own[i].pages[-1] for i in copies], self._free[-len(copies):].tolist()
            copy_pages(self.pool, src, dst)
            del self._free[-len(copies):]
            for i, p, q in zip(copies, src, dst):
                self._users[p] -= 1
                self._users[q] = 1
                own[i].pages[-1] = q
        for s, c in zip(own, counts):
            s.length += c
            while len(s.pages) * self.page < s.length:
                p = self._free.pop()
                self._users[p] = 1
                s.pages.append(p)
        try:
            return self._batch(own, counts)
        except BaseException:
            for s, c in zip(own, counts):
                self._cut(s, s.length - c)
            raise

    def _batch(self, own, counts) -> Batch:
        """The batch's arrays, in one copy to the device."""
        width, n = max([len(s.pages) for s in own], default=0), len(own)
        flat = array("i", [s.length for s in own])
        at = 0
        flat.append(0)
        for c in counts:
            at += c
            flat.append(at)
        for s in own:
            flat.extend(s.pages)
            flat.extend(array("i", [-1]) * (width - len(s.pages)))
        host = torch.frombuffer(flat, dtype=torch.int32)
        if self.pool.is_cuda:  # (from pinned memory: a copy from other memory waits for the stream)
            host = torch.empty(host.shape, dtype=torch.int32, pin_memory=True).copy_(host)
        dev = host.to(self.pool.device, non_blocking=True)
        return Batch(dev[2 * n + 1:].view(n, width), dev[:n], dev[n:2 * n + 1], counts)

    def compact(self) -> int:
        """Moves pages so that those in use are the first of the pool (which a caller may then copy into a smaller one);
        their number.  Batches given out before are no longer valid."""
        self._refuse_capture("compact")
        used = len(self._users) - len(self._free)
        holes = [p for p in range(used) if self._users[p] == 0]
        moved = [p for p in range(used, len(self._users)) if self._users[p] > 0]
        if moved:
            copy_pages(self.pool, moved, holes)
            to = dict(zip(moved, holes))
            for p, q in to.items():
                self._users[q], self._users[p] = self._users[p], 0
            for s in self._sequences.values():
                s.pages = array("i", [to.get(p, p) for p in s.pages])
        self._free = array("i", range(len(self._users) - 1, used - 1, -1))
        return used
