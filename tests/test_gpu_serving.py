"""The operators of serving from a cache (ethos_amd.serving) against float64.  Tolerances count
roundings: u(T) = finfo(T).eps / 2 for a value stored in T, U = 2^-24 for a float32 operation."""
import math

import pytest
import torch

import ethos_amd
from ethos_amd import hip

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
half_step = lambda dt: torch.finfo(dt).eps / 2  # noqa: E731
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rates(rope):
    return 1.0 / 10000.0 ** (torch.arange(0, rope, 2, device="cuda", dtype=torch.float32) / max(1, rope))


def _turned(r, pos, rates):
    """[..., rope] rows at positions [n], float64."""
    t = pos.double()[:, None] * rates.double()
    t = t.view(len(pos), *([1] * (r.dim() - 2)), len(rates))
    a, b = r.double().chunk(2, -1)
    return torch.cat((a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()), -1)


def _layout(lens, page, seed=0, extra=3, width=None):
    """(table, number of pages): scattered pages for sequences of these lengths, -1 behind them."""
    g = _gen(seed + 99)
    each = [-(-n // page) for n in lens]
    total = sum(each) + extra
    numbers = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width or max(each + [1]) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, k in enumerate(each):
        table[i, :k] = numbers[at:at + k]
        at += k
    return table, total


def _starts(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return i32(s)


def _slots(table, i, pos, page):
    return table[i].long()[pos // page] * page + pos % page


def _within(got, want, bound, what):
    d = (got.double() - want).abs()
    bad = ~(d <= bound + 1e-30)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((d / (bound + 1e-30)).max()):.3g} bounds"


# ------------------------------------------------------------------------------- append
APPEND = [  # (lens, new, rank, rope, page)
    ([1], [1], 256, 64, 64),
    ([5, 64, 65, 1], [5, 1, 2, 1], 256, 64, 64),
    ([300, 7, 100000], [33, 0, 7], 128, 32, 16),
    ([17, 40], [17, 3], 512, 128, 1),
    ([1000], [257], 8, 8, 4),
]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,new,rank,rope,page", APPEND)
def test_append_against_float64(lens, new, rank, rope, page, dt):
    g, T = _gen(rank + len(lens)), DT[dt]
    table, pages = _layout(lens, page)
    n = sum(new)
    wide = (torch.randn(n + 2, 16 + rank + rope, generator=g, device="cuda") * torch.rand(n + 2, 1, generator=g, device="cuda") * 3).to(T)
    rows = wide[:, 16:]
    gain = (1 + 0.2 * torch.randn(rank, generator=g, device="cuda")).to(T)
    pool = torch.full((pages, page, rank + rope), 7.0, dtype=T, device="cuda")
    version = pool._version
    ethos_amd.latent_append(rows, gain, pool, table, i32(lens), _starts(new), _rates(rope), eps=1e-6)
    assert pool._version > version
    want = torch.full((pages * page, rank + rope), 7.0, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    at = 0
    for i, (length, m) in enumerate(zip(lens, new)):
        x = rows[at:at + m].double()
        at += m
        pos = torch.arange(length - m, length, device="cuda")
        y = x[:, :rank] * torch.rsqrt(x[:, :rank].square().mean(1, keepdim=True) + 1e-6) * gain.double()
        k = _turned(x[:, rank:], pos, _rates(rope))
        size = (x[:, rank:].abs().view(m, 2, rope // 2).sum(1)).repeat(1, 2)  # |a| + |b|
        slot = _slots(table, i, pos, page)
        want[slot] = torch.cat((y, k), 1)
        # the mean's sum, its root and three products; the angle is off by 2^-24 pi, its cosine and sine by two steps
        bound[slot] = torch.cat((y.abs() * (rank + 16) * U, size * 10 * U), 1) + half_step(T) * want[slot].abs() * 1.01
    _within(pool.view(-1, rank + rope), want, bound, "pool")


def test_append_leaves_out_what_has_no_place():
    rank, rope, page = 16, 8, 4
    rows = torch.randn(9, rank + rope, device="cuda")
    gain = torch.ones(rank, device="cuda")
    pool = torch.zeros(6, page, rank + rope, device="cuda")
    # pages outside the pool; a length beyond the table; more new tokens than the length; a negative length
    table = i32([[0, 6], [2, 3], [-1, 1], [4, 5]])
    ethos_amd.latent_append(rows, gain, pool, table, i32([6, 10, 6, 1]), i32([0, 2, 4, 7, 9]), _rates(rope))
    filled = (pool.abs().sum(-1) > 0).view(-1).nonzero()[:, 0].tolist()
    # sequence 2: positions 3, 4, 5, of which 4 and 5 are in page 1; sequence 3: positions -1 and 0, in page 4
    assert filled == [4, 5, 16]
    pool.zero_()
    ethos_amd.latent_append(rows, gain, pool, table[:1], i32([-3]), i32([0, 9]), _rates(rope))
    ethos_amd.latent_append(rows, gain, pool, table[:1], i32([0]), i32([0, 0]), _rates(rope))
    ethos_amd.latent_append(rows, gain, pool, table[:0], i32([]), i32([0]), _rates(rope))
    ethos_amd.latent_append(rows[:0], gain, pool, table[:1], i32([4]), i32([0, 0]), _rates(rope))
    ethos_amd.latent_append(rows, gain, pool, table[:, :0], i32([4, 4, 4, 4]), i32([0, 2, 4, 7, 9]), _rates(rope))
    assert float(pool.abs().sum()) == 0.0


def test_append_of_more_rows_than_a_launch_has_threads_for():
    """2^26 rows and some, of two sequences."""
    n, page, first, g = (1 << 26) + 7, 65536, (1 << 25) + 12345, _gen(24)
    rows = (torch.randn(n, 8, generator=g, device="cuda") * 2).to(torch.bfloat16)
    gain = (1 + 0.2 * torch.randn(8, generator=g, device="cuda")).to(torch.bfloat16)
    width = -(-(n - first) // page) + 1
    table = torch.randperm(2 * width, generator=g, device="cuda").to(torch.int32).view(2, width)
    pool = torch.full((2 * width, page, 8), 7.0, dtype=torch.bfloat16, device="cuda")
    ethos_amd.latent_append(rows, gain, pool, table, i32([first, n - first]), i32([0, first, n]), _rates(0), eps=1e-6)
    for i, (a, z) in enumerate(((0, first), (first, n))):
        whole = pool[table[i].long()].view(-1, 8)  # the sequence's rows in order
        for r0 in range(a, z, 1 << 24):
            x = rows[r0:min(z, r0 + (1 << 24))].double()
            want = x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-6) * gain.double()
            _within(whole[r0 - a:r0 - a + len(x)], want, want.abs() * (24 * U + half_step(torch.bfloat16) * 1.01), f"rows from {r0}")
        assert bool((whole[z - a:] == 7.0).all())


# ------------------------------------------------------------------------------- attention
def _case(lens, new, H, rank, rope, nope, v, page, dt, seed=0, extra=3, size=1.5):
    g, T = _gen(seed), DT[dt]
    table, pages = _layout(lens, page, seed, extra)
    pool = torch.full((pages, page, rank + rope), math.nan, dtype=T, device="cuda")
    flat = pool.view(-1, rank + rope)
    for i, n in enumerate(lens):
        flat[_slots(table, i, torch.arange(n, device="cuda"), page)] = torch.randn(n, rank + rope, generator=g, device="cuda").to(T)
    w = (torch.randn(H * (nope + v), rank, generator=g, device="cuda") / math.sqrt(rank)).to(T)
    q = (torch.randn(sum(new), H, nope + rope, generator=g, device="cuda") * size).to(T)
    return dict(q=q, w=w, pool=pool, table=table, lens=i32(lens), starts=_starts(new), rates=_rates(rope), scale=1 / math.sqrt(nope + rope))


def _attend(c, **kw):
    return ethos_amd.paged_attention(c["q"], c["w"], c["pool"], c["table"], c["lens"], c["starts"], c["rates"], c["scale"], **kw)


def _oracle(c):
    """(out, bound, score size) in float64.  A score's terms: the query times the weight, (nope + 2) U of their sizes
    and its rounding u, times the row, another (rank + rope + 8) U; exponentials are off by as much as
    their scores and (bf16) a rounding, the weighted latents by both, their sums' additions and a rounding,
    the result by the rank's additions and its rounding."""
    q, w, T = c["q"].double(), c["w"].double(), c["q"].dtype
    n, H, qw = q.shape
    rank = w.shape[1]
    rope = c["pool"].shape[2] - rank
    nope = qw - rope
    w = w.view(H, -1, rank)
    page = c["pool"].shape[1]
    t = half_step(T) if T == torch.bfloat16 else 0.0
    out = torch.full((n, H, w.shape[1] - nope), math.nan, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    flat = c["pool"].view(-1, rank + rope).double()
    starts = c["starts"].tolist()
    spread = 0.0
    for i, length in enumerate(c["lens"].tolist()):
        a, z = starts[i], starts[i + 1]
        if z == a:
            continue
        rows = flat[_slots(c["table"], i, torch.arange(length, device="cuda"), page)]
        first = length - (z - a)
        pos = torch.arange(first, length, device="cuda")
        seen = torch.arange(length, device="cuda")[None, :] <= pos[:, None]
        for h in range(H):
            turn = _turned(q[a:z, h, nope:], pos, c["rates"])
            wide = torch.cat((q[a:z, h, :nope] @ w[h, :nope], turn), 1)
            pair = q[a:z, h, nope:].abs().view(z - a, 2, -1).sum(1).repeat(1, 2)
            sizes = torch.cat((q[a:z, h, :nope].abs() @ w[h, :nope].abs(), pair), 1)
            s = (wide @ rows.T * c["scale"]).masked_fill(~seen, -math.inf)
            e_s = sizes @ rows.abs().T * c["scale"] * (t + (nope + rank + rope + 32) * U) + 8 * U * s.abs().nan_to_num(0, 0, 0)
            e_s = torch.where(seen, e_s, torch.zeros_like(e_s)).amax(1, keepdim=True)
            p = torch.softmax(s, 1)
            spread = max(spread, float(s[-1].isfinite().sum() > 1 and s[-1][s[-1].isfinite()].std()))
            lat, big = p @ rows[:, :rank], p @ rows[:, :rank].abs()
            e_lat = big * (torch.expm1(2 * e_s) + 2 * t + (length + 64) * U)
            o = lat @ w[h, nope:].T
            out[a:z, h] = o
            bound[a:z, h] = (e_lat + lat.abs() * t) @ w[h, nope:].abs().T + (rank + 8) * U * (lat.abs() @ w[h, nope:].abs().T) \
                + half_step(T) * o.abs() * 1.01 + 1e-30
    return out.view(n, -1), bound.view(n, -1), spread


def _near(got, c, what=""):
    """Within the bounds, and in the 2-norm within twice what independent roundings leave: the result's, the latents', the
    exponentials' and the score's, whose queries' rounding of u / sqrt(3) weighs as much as scores spread."""
    want, bound, spread = _oracle(c)
    rows = ~want.isnan().any(1)
    _within(got[rows], want[rows], bound[rows], what)
    u = half_step(c["q"].dtype)
    limit = 2 * u / math.sqrt(3) * math.sqrt(3 + 2 * spread ** 2) if c["q"].dtype == torch.bfloat16 else 128 * U
    err = float((got[rows].double() - want[rows]).norm() / want[rows].norm())
    assert err <= limit, f"{what}: normalised error {err:.3e} above {limit:.3e}"


ATTEND = [  # (lens, new, H, rank, rope, nope, v, page)
    ([1], [1], 16, 256, 64, 64, 64, 64),
    ([64], [1], 16, 256, 64, 64, 64, 64),
    ([65], [1], 16, 256, 64, 64, 64, 64),
    ([1000, 1, 63, 4097, 128], [1, 1, 1, 1, 1], 16, 256, 64, 64, 64, 64),
    ([777, 300, 20, 64], [5, 1, 3, 0], 16, 256, 64, 64, 64, 16),
    ([130, 700], [130, 257], 16, 256, 64, 64, 64, 128),
    ([200, 91, 90], [9, 91, 2], 4, 256, 64, 64, 64, 1),
    ([513], [200], 12, 256, 64, 64, 64, 256),
    ([90, 2000], [7, 1], 32, 256, 64, 64, 64, 32),
    ([350], [3], 1, 256, 64, 64, 64, 2),
    ([50, 129, 5], [50, 1, 5], 3, 256, 64, 64, 64, 8),
    ([300, 65], [20, 2], 8, 256, 64, 128, 32, 64),
    ([100, 7], [3, 7], 4, 32, 16, 16, 16, 16),
    ([100, 260], [1, 33], 2, 512, 128, 24, 40, 64),
    ([30], [2], 3, 8, 8, 5, 3, 4),
]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,new,H,rank,rope,nope,v,page", ATTEND)
def test_attention_against_float64(lens, new, H, rank, rope, nope, v, page, dt):
    c = _case(lens, new, H, rank, rope, nope, v, page, dt, seed=sum(lens) + H)
    got = _attend(c)
    _near(got, c, f"{lens} {new}")
    assert torch.equal(_attend(c), got)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_attention_of_one_position_is_its_value(dt):
    c = _case([1, 1], [1, 1], 16, 256, 64, 64, 64, 64, dt)
    rows = torch.stack([c["pool"][int(c["table"][i, 0]), 0, :256] for i in range(2)]).double()
    v = rows @ c["w"].double().view(16, 128, 256)[:, 64:].reshape(-1, 256).T
    size = rows.abs() @ c["w"].double().view(16, 128, 256)[:, 64:].reshape(-1, 256).abs().T
    # a weight of exactly one: the latents are exact
    _within(_attend(c), v, half_step(DT[dt]) * v.abs() * 1.01 + size * 270 * U, "value")


@pytest.mark.parametrize("dt,rank", [("bf16", 256), ("bf16", 64), ("fp32", 64)])
def test_attention_sees_nothing_behind_a_token(dt, rank):
    """NaN and infinities in later tokens of the same chunk, in unused places and in other sequences' pages."""
    lens, new = [150, 40, 333], [37, 40, 9]
    c = _case(lens, new, 4, rank, 64, 64, 64, 16, dt, seed=3)
    want = _attend(c)
    flat = c["pool"].view(-1, rank + 64)
    starts = c["starts"].tolist()
    for cut, value in ((5, math.nan), (1, math.inf), (8, -math.inf)):
        for i in range(3):
            spoiled = torch.arange(lens[i] - cut, lens[i], device="cuda")
            keep = flat[_slots(c["table"], i, spoiled, 16)].clone()
            flat[_slots(c["table"], i, spoiled, 16)] = value
            got = _attend(c)
            flat[_slots(c["table"], i, spoiled, 16)] = keep
            hit = torch.zeros(len(got), dtype=torch.bool, device="cuda")
            hit[starts[i + 1] - cut:starts[i + 1]] = True
            assert torch.equal(got[~hit], want[~hit]), (cut, value, i)
            assert bool(got[hit].isnan().all()), (cut, value, i)


def test_many_new_tokens_see_nothing_behind_them():
    """The same where keys and values are formed first."""
    lens, new = [450, 200, 1000], [300, 200, 131]
    c = _case(lens, new, 3, 256, 64, 64, 64, 32, "bf16", seed=13)
    want = _attend(c)
    _near(want, c)
    flat = c["pool"].view(-1, 320)
    starts = c["starts"].tolist()
    for cut, value in ((5, math.nan), (1, math.inf), (100, -math.inf)):
        for i in range(3):
            spoiled = _slots(c["table"], i, torch.arange(lens[i] - cut, lens[i], device="cuda"), 32)
            keep = flat[spoiled].clone()
            flat[spoiled] = value
            got = _attend(c)
            flat[spoiled] = keep
            hit = torch.zeros(len(got), dtype=torch.bool, device="cuda")
            hit[starts[i + 1] - cut:starts[i + 1]] = True
            assert torch.equal(got[~hit], want[~hit]), (cut, value, i)
            assert bool(got[hit].isnan().all()), (cut, value, i)


def test_many_new_tokens_of_batches_that_do_not_fit():
    c = _case([400, 333, 150], [200, 150, 140], 4, 256, 64, 64, 64, 16, "bf16", seed=14)
    good = _attend(c)
    out = torch.full((500, 256), 5.0, dtype=torch.bfloat16, device="cuda")
    c["q"] = torch.cat((c["q"], c["q"][:10] * math.nan))
    got = _attend(c, out=out)
    assert torch.equal(got[:490], good) and bool((got[490:] == 5.0).all())
    table = c["table"].clone()
    c["table"] = table.clone()
    c["table"][1, 15] = 10 ** 8  # positions 240 to 255, the first of them seen by all but 57 of the new tokens
    got = _attend(c)
    assert bool(got[200 + 57:350].isnan().all()) and torch.equal(got[:257], good[:257]) and torch.equal(got[350:490], good[350:])
    c["table"] = table
    for length in (16 * table.shape[1] + 1, 2 ** 31 - 1, 2 ** 30 + 1, -1, -2 ** 31):
        c["lens"] = i32([400, length, 150])
        got = _attend(c)
        assert bool(got[200:350].isnan().all()) and torch.equal(got[:200], good[:200]) and torch.equal(got[350:490], good[350:]), length
    c["lens"] = i32([400, 3, 150])  # three positions: the first 147 tokens see none
    got = _attend(c)
    assert float(got[200:347].float().abs().sum()) == 0.0 and not bool(got[347:350].isnan().any()) and bool((got[347:350] != 0).any())
    assert torch.equal(got[350:490], good[350:])
    c["lens"] = i32([400, 333, 150])
    c["starts"] = i32([0, 200, 350, 4000])
    got = _attend(c)
    assert torch.equal(got[:350], good[:350]) and bool(got[350:].isnan().all())
    c["starts"] = i32([0, 490, 0, 490])  # sequences that overlap
    _attend(c)
    c["starts"] = i32([0, 0, 0, 140])
    c["q"], c["lens"] = c["q"][350:], i32([400, 333, 150])
    out = torch.full((150, 256), 5.0, dtype=torch.bfloat16, device="cuda")
    got = _attend(c, out=out)
    assert bool((got[140:] == 5.0).all())
    _near(got, c, "50 tokens a sequence on the average")  # (fewer than the form of `good` is for)


@pytest.mark.parametrize("lens,new,H,page", [([128], [128], 1, 8), ([129], [129], 5, 64), ([5000], [128], 2, 64), ([300, 300, 300], [129, 254, 1], 16, 16),
                                             ([2000, 700], [1100, 511], 8, 512), ([600, 1, 90], [600, 1, 0], 7, 8)])
def test_many_new_tokens_against_float64(lens, new, H, page):
    c = _case(lens, new, H, 256, 64, 64, 64, page, "bf16", seed=sum(new))
    got = _attend(c)
    _near(got, c, f"{lens} {new}")
    assert torch.equal(_attend(c), got)


@pytest.mark.parametrize("dt,rank", [("bf16", 256), ("fp32", 64)])
@pytest.mark.parametrize("singles,drafts,idle", [(3, 1, 0), (8, 0, 2), (20, 4, 0), (60, 0, 5), (1, 0, 30)])
def test_chunks_beside_single_tokens_against_float64(singles, drafts, idle, dt, rank):
    """A chunk of a prompt, a shorter one, single tokens, a few drafted ones and sequences without new tokens in one batch: with 96 and
    more new tokens a sequence on the average, and with fewer."""
    new = [1] * singles + [700] + [5] * drafts + [0] * idle + [300]
    lens = [1 + (i * 613) % 1500 for i in range(singles)] + [1200] + [5 + 77 * i for i in range(drafts)] + [200] * idle + [300]
    c = _case(lens, new, 4, rank, 64, 64, 64, 32, dt, seed=singles)
    got = _attend(c)
    _near(got, c, f"{singles} {drafts} {idle}")
    assert torch.equal(_attend(c), got)


@pytest.mark.parametrize("new", [1, 150])
@pytest.mark.parametrize("of_rows,of_weight,of_query", [(64.0, 16.0, 1.0), (2.0 ** -6, 2.0 ** -3, 1.0), (1.0, 1.0, 2.0 ** 10), (1.0, 1.0, 2.0 ** -8),
                                                        (2.0 ** -4, 2.0 ** 10, 2.0 ** -4)])
def test_attention_of_other_magnitudes(new, of_rows, of_weight, of_query):
    """Rows, weights and queries times powers of two, with scores as before: the same relative bounds."""
    c = _case([400, 170], [new, new], 4, 256, 64, 64, 64, 16, "bf16", seed=new)
    c["w"] = c["w"] * of_weight
    rank = c["w"].shape[1]
    c["pool"][..., :rank] *= of_rows
    c["pool"][..., rank:] *= of_rows * of_weight
    c["q"] = c["q"] * of_query
    c["scale"] /= of_rows * of_weight * of_query
    _near(_attend(c), c, f"{new} new")


def test_keys_and_values_out_of_range_count_as_infinite():
    """Many new tokens: a finite row whose values do not fit has no result where it is seen, and does not show elsewhere."""
    c = _case([300, 200], [200, 150], 4, 256, 64, 64, 64, 16, "bf16", seed=3)
    good = _attend(c)
    at = _slots(c["table"], 0, torch.tensor([250], device="cuda"), 16)
    c["pool"].view(-1, 320)[at] = 1e36
    got = _attend(c)
    assert torch.equal(got[:150], good[:150]) and torch.equal(got[200:], good[200:])
    assert bool(got[150:200].isnan().all())


@pytest.mark.parametrize("dt,rank", [("bf16", 256), ("bf16", 64), ("fp32", 64)])
def test_attention_of_batches_that_do_not_fit(dt, rank):
    c = _case([70, 33, 100, 20], [3, 2, 4, 2], 4, rank, 64, 64, 64, 16, dt, seed=4)
    good = _attend(c)
    out = torch.full((13, good.shape[1]), 5.0, dtype=DT[dt], device="cuda")
    c["q"] = torch.cat((c["q"], c["q"][:2] * math.nan))
    # rows behind the last sequence stay
    got = _attend(c, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got[:11], good) and bool((got[11:] == 5.0).all())
    # a page outside the pool: NaN for the tokens that see it
    table = c["table"].clone()
    c["table"] = table.clone()
    c["table"][2, 6] = 10 ** 6  # positions 96 to 99
    got = _attend(c)
    assert bool(got[5:9].isnan().all()) and torch.equal(got[:5], good[:5]) and torch.equal(got[9:11], good[9:])
    c["table"][2, 6] = table[2, 6]
    c["table"][2, 0] = -5
    got = _attend(c)
    assert bool(got[5:9].isnan().all()) and torch.equal(got[9:11], good[9:])
    c["table"] = table
    # lengths beyond the table or negative: NaN; fewer positions than new tokens: the first tokens see nothing
    for length in (16 * table.shape[1] + 1, 2 ** 31 - 1, -1, -2 ** 31):
        c["lens"] = i32([70, 33, length, 20])
        got = _attend(c)
        assert bool(got[5:9].isnan().all()) and torch.equal(got[:5], good[:5]) and torch.equal(got[9:11], good[9:]), length
    c["lens"] = i32([70, 33, 1, 20])
    got = _attend(c)
    assert float(got[5:8].float().abs().sum()) == 0.0 and not bool(got[8].isnan().any()) and torch.equal(got[9:11], good[9:])
    c["lens"] = i32([70, 33, 0, 20])
    assert float(_attend(c)[5:9].float().abs().sum()) == 0.0
    c["lens"] = i32([70, 33, 100, 20])
    # starts that leave the batch or run backwards: those rows NaN or untouched, the others right
    c["starts"] = i32([0, 3, 5, 9, 40])
    got = _attend(c)
    assert torch.equal(got[:9], good[:9]) and bool(got[9:].isnan().all())
    c["starts"] = i32([0, 3, 5, 2, 11])
    assert torch.equal(_attend(c)[:2], good[:2])
    # nothing to do
    c["starts"], c["q"] = i32([0, 0, 0, 0, 0]), c["q"][:0]
    assert _attend(c).shape == (0, good.shape[1])


@pytest.mark.parametrize("dt,rank", [("bf16", 256), ("fp32", 32)])
def test_attention_takes_views_and_shared_pages(dt, rank):
    c = _case([200, 200], [6, 6], 4, rank, 64, 64, 64, 16, dt, seed=5)
    c["table"][1, :10] = c["table"][0, :10]  # a fork: ten pages in common
    got = _attend(c)
    _near(got, c, "shared pages")
    wide = torch.full((2, 40), -7, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + c["table"].shape[1]] = c["table"]
    c["table"] = wide[:, 3:3 + c["table"].shape[1]]
    assert torch.equal(_attend(c), got)
    flat = torch.empty(c["q"].numel() + 3, dtype=DT[dt], device="cuda")
    flat[3:] = c["q"].reshape(-1)
    c["q"] = flat[3:].view(c["q"].shape)  # an address that is no multiple of 16
    assert torch.equal(_attend(c), got)


def test_attention_over_a_pool_beyond_32_bits():
    """Pages whose offset passes 2^32 bytes."""
    page, pages = 64, 110000  # 4.5 GB
    c = _case([500, 100], [3, 1], 16, 256, 64, 64, 64, page, "bf16", seed=6)
    want = _attend(c)
    pool = torch.zeros(pages, page, 320, dtype=torch.bfloat16, device="cuda")
    far = torch.randperm(2000, generator=_gen(1), device="cuda")[:c["pool"].shape[0]] + (pages - 2000)
    pool[far] = c["pool"]
    c["table"] = torch.where(c["table"] >= 0, far[c["table"].long().clamp(min=0)].to(torch.int32), c["table"])
    c["pool"] = pool
    assert torch.equal(_attend(c), want)
    rows = torch.randn(4, 320, device="cuda").to(torch.bfloat16)
    small = torch.zeros(1, 64, 320, dtype=torch.bfloat16, device="cuda")
    gain = torch.ones(256, dtype=torch.bfloat16, device="cuda")
    ethos_amd.latent_append(rows, gain, small, i32([[0]]), i32([9]), i32([0, 4]), c["rates"])
    ethos_amd.latent_append(rows, gain, pool, i32([[pages - 1]]), i32([9]), i32([0, 4]), c["rates"])
    assert torch.equal(pool[-1, :16], torch.cat((torch.zeros_like(small[0, :5]), small[0, 5:9], torch.zeros_like(small[0, 9:16])))
                       .where(torch.arange(16, device="cuda")[:, None].lt(9) & torch.arange(16, device="cuda")[:, None].ge(5), pool[-1, :16]))
    blocks = pool.view(2, pages // 2, page, 320)
    ethos_amd.copy_pages(blocks, [pages // 2 - 1], [5])
    assert torch.equal(blocks[:, 5], blocks[:, -1])


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_attention_under_large_scores(dt):
    """Scores of hundreds: one key takes all the weight, no exponential overflows."""
    c = _case([300, 90], [4, 90], 16, 256, 64, 64, 64, 64, dt, seed=7, size=300.0)
    got = _attend(c)
    want, bound, _ = _oracle(c)
    assert bool(got.isfinite().all())
    sure = bound.isfinite() & (bound < 0.05)  # where two keys are near, the oracle says nothing
    assert not bool(((got.double() - want).abs() > bound)[sure].any())


@pytest.mark.parametrize("dt,rank,new", [("bf16", 256, 3), ("bf16", 256, 150), ("bf16", 64, 3), ("fp32", 64, 40)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_attention_over_infinite_rotary_keys(dt, rank, new, sign):
    """An infinite value in a cached key alone: a score of +inf leaves no result, one of -inf no weight (or, of a query that goes into the
    products as two values, no result); scores of -inf everywhere leave none.  (With rates of zero, so that a query keeps its signs.)"""
    c = _case([400, 170], [new, new], 4, rank, 64, 64, 64, 16, dt, seed=21)
    c["rates"] = torch.zeros_like(c["rates"])
    c["q"][:, :2, 64 + 5] = c["q"][:, :2, 64 + 5].abs() * sign + 0.25 * sign  # heads 0 and 1 towards +inf, 2 and 3 to -inf
    c["q"][:, 2:, 64 + 5] = c["q"][:, 2:, 64 + 5].abs() * -sign - 0.25 * sign
    good = _attend(c)
    _near(good, c)
    flat = c["pool"].view(-1, rank + 64)
    at = _slots(c["table"], 0, torch.tensor([200], device="cuda"), 16)
    flat[at, rank + 5] = sign * math.inf
    got = _attend(c)
    assert torch.equal(got[new:], good[new:])
    heads = got.view(-1, 4, 64)
    assert bool(heads[:new, :2].isnan().all())
    split = dt == "bf16" and rank == 256 and new < 96
    # the same without that position
    rest = dict(c, pool=c["pool"].clone(), lens=i32([399, 170]))
    p = torch.arange(400, device="cuda")
    rest["pool"].view(-1, rank + 64)[_slots(c["table"], 0, p[:399], 16)] = flat[_slots(c["table"], 0, p[p != 200], 16)]
    want, bound, _ = _oracle(rest)
    far = (heads.double() - want.view(heads.shape)).abs() > bound.view(heads.shape)
    none = heads.isnan()
    assert not bool((far & ~none)[:new, 2:].any()) and (split or not bool(none[:new, 2:].any()))
    # one that the last token alone sees
    keep = flat[_slots(c["table"], 0, p, 16), rank + 5].clone()
    keep[200] = 0.5
    flat[_slots(c["table"], 0, p, 16), rank + 5] = keep
    good[:new] = _attend(c)[:new]
    flat[_slots(c["table"], 0, p[399:], 16), rank + 5] = sign * math.inf
    got = _attend(c)
    assert torch.equal(got[:new - 1], good[:new - 1]) and torch.equal(got[new:], good[new:])
    assert bool(got.view(-1, 4, 64)[new - 1, :2].isnan().all())
    # every position
    flat[_slots(c["table"], 0, p, 16), rank + 5] = sign * math.inf
    got = _attend(c)
    assert torch.equal(got[new:], good[new:]) and bool(got[:new].isnan().all())


@pytest.mark.parametrize("dt,rank,new", [("bf16", 256, 2), ("bf16", 256, 130), ("bf16", 64, 2), ("fp32", 64, 40)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_attention_under_scores_far_from_zero(dt, rank, new, sign):
    """Scores of up to 2^20 to 2^100 (2^36 with many new tokens, whose keys have a range) at one position, at half of that or less,
    or twice as far below zero, at the others: the value at that position.  In the rotary columns alone, which rates of zero leave."""
    lens, at = [333, 170], [210, 5]
    for exponent in (10, 20, 24, 26, 27, 28, 29, 30, 31, 32, 33, 36, 50, 100)[:12 if new > 96 else None]:
        c = _case(lens, [new, new], 4, rank, 64, 64, 64, 16, dt, seed=exponent)
        c["rates"] = torch.zeros_like(c["rates"])
        g = _gen(exponent)
        # a query of `size` times a number in (1, 1.9) a row, along a key of as much, 64 columns: no power of two anywhere
        size = math.sqrt(2.0 ** exponent / 64 / c["scale"])
        u = 1.0 + 0.2 * torch.rand(64, generator=g, device="cuda")
        far = 1.0 + 0.9 * torch.rand(2 * new, 4, 1, generator=g, device="cuda")
        c["q"] = torch.cat((torch.zeros(2 * new, 4, 64, device="cuda"), far * size * u), -1).to(DT[dt])
        flat = c["pool"].view(-1, rank + 64)
        want = []
        for i in range(2):
            slots = _slots(c["table"], i, torch.arange(lens[i], device="cuda"), 16)
            part = torch.rand(lens[i], 1, generator=g, device="cuda") * 0.5 if sign > 0 else -2.0 - torch.rand(lens[i], 1, generator=g, device="cuda")
            part[at[i]] = sign
            flat[slots, rank:] = (part * size * u).to(DT[dt])
            row = flat[slots[at[i]], :rank].double()
            w = c["w"].double().view(4, 128, rank)[:, 64:]
            for pos in range(lens[i] - new, lens[i]):
                want.append(((w @ row).reshape(-1), (w.abs() @ row.abs()).reshape(-1)) if pos >= at[i] else None)
        got = _attend(c)
        assert bool(got.isfinite().all()), exponent
        for k, x in enumerate(want):
            if x is not None:
                # the row's rounding as an operand and the result's, and those of its parts' join
                _within(got[k], x[0], x[1] * (2 * (half_step(DT[dt]) if dt == "bf16" else 0.0) + (rank + 64) * U) + half_step(DT[dt]) * x[0].abs() * 1.01,
                        f"2^{exponent}, row {k}")


@pytest.mark.parametrize("dt,rank,new", [("bf16", 256, 3), ("bf16", 256, 150), ("fp32", 64, 3)])
def test_attention_under_the_largest_and_smallest_scales(dt, rank, new):
    """Scores of zero at 1e35, and a scale that leaves no differences: the mean of the values that a token sees."""
    for scale in (1e35, 1e-38):
        c = _case([200, 170], [new, new], 4, rank, 64, 64, 64, 16, dt, seed=22)
        if scale > 1:
            c["q"] = torch.zeros_like(c["q"])
        c["scale"] = scale
        _near(_attend(c), c, str(scale))
    with pytest.raises(RuntimeError, match="1e35"):
        _attend(dict(c, scale=2e35))


@pytest.mark.parametrize("new", [1, 6, 64])
@pytest.mark.parametrize("middle", [1, 333])
def test_attention_in_streams_and_graphs(new, middle):
    a = _case([900, 333, 64], [new, middle, new], 16, 256, 64, 64, 64, 64, "bf16", seed=8)
    b = _case([64, 2000, 90], [new, middle, new], 16, 256, 64, 64, 64, 64, "bf16", seed=9)
    want = [_attend(a), _attend(b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, c in zip(streams, (a, b)):
        with torch.cuda.stream(s):
            got.append([_attend(c) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for xs, w in zip(got, want) for x in xs)
    # two captured calls, replayed in turn with eager work between, over inputs that change
    static = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    pages = max(a["pool"].shape[0], b["pool"].shape[0])
    static["pool"] = torch.zeros(pages, 64, 320, dtype=torch.bfloat16, device="cuda")
    width = max(a["table"].shape[1], b["table"].shape[1])
    static["table"] = torch.full((3, width), -1, dtype=torch.int32, device="cuda")
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _attend(static)
    with torch.cuda.graph(other):
        out2 = _attend(static)
    for k in range(6):
        c, w = (a, want[0]) if k % 2 == 0 else (b, want[1])
        for name in ("q", "w", "lens", "starts", "rates"):
            static[name].copy_(c[name])
        static["pool"][: c["pool"].shape[0]] = c["pool"]
        static["table"].fill_(-1)
        static["table"][:, : c["table"].shape[1]] = c["table"]
        (graph if k % 3 else other).replay()
        eager = _attend(c)
        torch.cuda.synchronize()
        assert torch.equal(out if k % 3 else out2, w) and torch.equal(eager, w), k


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_attention_of_more_rows_than_a_launch_has_threads_for(dt):
    """16,385 tokens of 1,024 heads: 2^24 rows and some."""
    n, H, g, T = 16385, 1024, _gen(23), DT[dt]
    pool = torch.randn(2, 4, 8, generator=g, device="cuda").to(T)
    w = torch.randn(H * 2, 8, generator=g, device="cuda").to(T) / 3
    q = torch.randn(n, H, 1, generator=g, device="cuda").to(T)
    lens = torch.randint(1, 9, (n,), generator=g, device="cuda").to(torch.int32)
    table = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda").repeat(n, 1)
    got = ethos_amd.paged_attention(q, w, pool, table, lens, torch.arange(n + 1, dtype=torch.int32, device="cuda"), _rates(0), 0.7)
    rows = pool.view(8, 8).double()
    k, v = rows @ w.double().view(H, 2, 8)[:, 0].T, rows @ w.double().view(H, 2, 8)[:, 1].T  # [8, H]
    size = rows.abs() @ w.double().abs().view(H, 2, 8)[:, 0].T
    for t0 in range(0, n, 4096):
        a = q[t0:t0 + 4096, :, 0].double()
        seen = torch.arange(8, device="cuda")[None, :, None] < lens[t0:t0 + 4096, None, None]
        s = (a[:, None, :] * k * 0.7).masked_fill(~seen, -math.inf)  # [., 8, H]
        want = (torch.softmax(s, 1) * v).sum(1)
        # float32 throughout: a score's terms are each off by some roundings, so is each weighted value's sum
        e = (a.abs()[:, None, :] * size * 0.7).amax(1) * 32 * U
        bound = (2 * e + 64 * U) * (rows.abs() @ w.double().abs().view(H, 2, 8)[:, 1].T).amax(0) + half_step(T) * want.abs() * 1.01
        _within(got[t0:t0 + 4096], want, bound, f"rows from {t0}")


# ------------------------------------------------------------------------------- pages
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("blocks,pages,page,width,pairs", [(1, 2, 1, 1, 1), (3, 40, 16, 320, 20), (2, 2000, 2, 24, 1000), (12, 9, 64, 320, 4),
                                                           (2, 1000, 1, 3, 451), (1, 5, 64, 320, 0)])
def test_copy_pages(blocks, pages, page, width, pairs, dt):
    pool = torch.randn(blocks, pages, page, width, generator=_gen(pages), device="cuda").to(DT[dt])
    at = torch.randperm(pages, generator=_gen(1), device="cuda").tolist()
    src, dst = at[:pairs], at[pairs:2 * pairs]
    if pairs > 4:
        src[3] = src[1]  # one page to several places
    want = pool.clone()
    if pairs:
        want[:, dst] = pool[:, src]
    version = pool._version
    ethos_amd.copy_pages(pool, src, torch.tensor(dst, dtype=torch.int64))
    assert torch.equal(pool, want) and pool._version > version


def test_copy_pages_in_a_graph():
    pool = torch.randn(3, 700, 8, 24, device="cuda")
    src, dst = list(range(0, 300)), list(range(350, 650))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ethos_amd.copy_pages(pool, src, dst)
    for _ in range(3):
        pool.normal_()
        want = pool.clone()
        want[:, dst] = pool[:, src]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool, want)


# ------------------------------------------------------------------------------- verification
def _verify_oracle(logits, drafts, u_accept, u_sample, probs, counts, temperature):
    """In float64 on the host, one sequence and one draft at a time."""
    z = logits.double().cpu()
    b, rows, V = z.shape
    accepted, tokens = [], []
    for i in range(b):
        n = rows - 1 if counts is None else max(0, min(rows - 1, int(counts[i])))
        if temperature:
            e = (z[i] - z[i].amax(-1, keepdim=True)) / temperature
            p = e.exp() / e.exp().sum(-1, keepdim=True)
        else:
            p = torch.nn.functional.one_hot(z[i].argmax(-1), V).double()
        took, rest = 0, None
        for j in range(n):
            x = int(drafts[i, j])
            q = torch.zeros(V, dtype=torch.float64) if probs is None else probs[i, j].double().cpu()
            if probs is None and 0 <= x < V:
                q[x] = 1.0
            if 0 <= x < V and float(u_accept[i, j]) * float(q[x]) < float(p[j, x]):
                took += 1
                continue
            rest = (p[j] - q).clamp(min=0)
            break
        if rest is None or not bool((rest > 0).any()):
            rest = p[took]
        up = rest.cumsum(0)
        accepted.append(took)
        above = (up > float(u_sample[i]) * float(up[-1])).nonzero()
        tokens.append(int(above[0]) if len(above) else int((rest > 0).nonzero()[-1]))
    return accepted, tokens


def _verify_case(b, m, V, dt, probs, seed, spread=2.5):
    g = _gen(seed)
    logits = (torch.randn(b, m + 1, V, generator=g, device="cuda") * spread).to(DT[dt])
    noisy = logits[:, :m].float() + torch.randn(b, m, V, generator=g, device="cuda") * 0.5
    p = torch.softmax(noisy, -1)
    drafts = torch.multinomial(p.view(-1, V), 1, generator=g).view(b, m) if m else torch.zeros(b, 0, dtype=torch.int64, device="cuda")
    u = torch.rand(b, m, generator=g, device="cuda"), torch.rand(b, generator=g, device="cuda")
    return logits, drafts, *u, None if probs == "none" else p.to(DT[probs])


@pytest.mark.parametrize("probs", ["fp32", "bf16", "none"])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("b,m,V", [(1, 0, 1), (3, 0, 777), (2, 1, 2), (5, 3, 100), (7, 4, 8191), (4, 2, 8193), (2, 9, 20001), (1, 255, 33),
                                   (200, 2, 6000), (1, 1, 2200000), (64, 4, 50000)])
def test_verify_against_float64(b, m, V, dt, probs):
    for temperature in (1.0, 0.6, 0.0):
        logits, drafts, ua, us, p = _verify_case(b, m, V, dt, probs, seed=b * 100 + V)
        counts = None if m == 0 else torch.randint(0, m + 1, (b,), generator=_gen(V), device="cuda").to(torch.int32)
        for c in (None, counts):
            got = ethos_amd.verify_drafts(logits, drafts, ua, us, draft_probs=p, counts=c, temperature=temperature)
            assert got[0].dtype == torch.int32 and got[1].dtype == torch.int64
            assert (got[0].tolist(), got[1].tolist()) == _verify_oracle(logits, drafts, ua, us, p, c, temperature)


def test_verify_at_the_edges_of_the_random_numbers():
    V = 9000
    logits, drafts, ua, us, p = _verify_case(6, 2, V, "fp32", "fp32", seed=1)
    logits[:, :, 0] = -math.inf   # no weight at either end
    logits[:, :, -1] = -math.inf
    for value in (0.0, 1.0 - 2.0 ** -24, 1.0, math.nan):
        us.fill_(value)
        ua.fill_(0.0 if value != value else value)
        got = ethos_amd.verify_drafts(logits, drafts, ua, us, draft_probs=p)
        if value == value:
            assert (got[0].tolist(), got[1].tolist()) == _verify_oracle(logits, drafts, ua, us, p, None, 1.0), value
        assert bool(((got[1] > 0) & (got[1] < V - 1)).all())


def test_verify_of_odd_inputs():
    V = 5000
    logits, drafts, ua, us, p = _verify_case(8, 2, V, "fp32", "fp32", seed=2)
    drafts[0, 0], drafts[1, 1], drafts[2, 0] = V, -1, 2 ** 62   # outside the vocabulary: not accepted
    ua[1, 0] = 0.0
    want = _verify_oracle(logits, drafts, ua, us, p, None, 1.0)
    got = ethos_amd.verify_drafts(logits, drafts, ua, us, draft_probs=p)
    assert (got[0].tolist(), got[1].tolist()) == want and want[0][0] == 0 and want[0][2] == 0
    # the draft's own probabilities equal to the model's, and a random number that refuses it all the same
    same = torch.softmax(logits[:, :2].double(), -1).float()
    ua.fill_(2.0)
    over = (same * 1.01).contiguous()  # nothing is left of p - q: drawn from p
    got = ethos_amd.verify_drafts(logits, drafts, ua, us, draft_probs=over)
    assert (got[0].tolist(), got[1].tolist()) == _verify_oracle(logits, drafts, ua, us, over, None, 1.0)
    # rows without a distribution
    ua.zero_()
    drafts = logits[:, :2].argmax(-1)
    logits[3, 0, 7] = math.nan
    logits[4, 1] = -math.inf
    logits[5, 2, 9] = math.inf
    logits[6, 2, 9] = math.nan
    got = ethos_amd.verify_drafts(logits, drafts, ua, us, draft_probs=p)
    assert got[0].tolist() == [2, 2, 2, 0, 1, 2, 2, 2] and (got[1] < 0).tolist() == [False] * 3 + [True] * 4 + [False]
    got = ethos_amd.verify_drafts(logits, drafts, ua, us, draft_probs=p, temperature=0.0)
    assert got[1].tolist()[3:7] == [-1, -1, 9, -1]
    counts = i32([-3, 0, 1, 2, 99, 0, 0, 0])  # outside [0, 2]: taken to the nearer end
    got = ethos_amd.verify_drafts(logits, drafts, ua, us, draft_probs=p, counts=counts)
    assert got[0].tolist() == [0, 0, 1, 0, 1, 0, 0, 0]
    assert ethos_amd.verify_drafts(logits[:0], drafts[:0], ua[:0], us[:0])[0].shape == (0,)


def test_verify_of_draft_probabilities_that_are_nan():
    """NaN in the row that the token is drawn with: no token.  In other rows it does not show."""
    V = 5000
    logits, _, ua, us, p = _verify_case(6, 2, V, "fp32", "fp32", seed=6)
    drafts = logits[:, :2].argmax(-1)
    ua.zero_()          # a draft of any weight stands
    ua[:4, 1] = 3e38    # ... but the second of these is refused
    good = ethos_amd.verify_drafts(logits, drafts, ua, us, draft_probs=p)
    assert good[0].tolist() == [1, 1, 1, 1, 2, 2] and bool((good[1] >= 0).all())
    p = p.clone()
    p[0, 1, 4999] = math.nan               # the refused draft's row
    p[1, 1, int(drafts[1, 1])] = math.nan  # ... at the draft itself
    p[2, 0, (int(drafts[2, 0]) + 1) % V] = math.nan  # the row of one that stands
    p[4, 1, (int(drafts[4, 1]) + 1) % V] = math.nan
    p[5, 0, int(drafts[5, 0])] = math.nan  # a draft of no known probability does not stand
    for many in (1, 90):  # (in one launch, in several)
        got = ethos_amd.verify_drafts(*[t.repeat(many, *[1] * (t.dim() - 1)) for t in (logits, drafts, ua, us)],
                                      draft_probs=p.repeat(many, 1, 1))
        assert got[0].tolist() == [1, 1, 1, 1, 2, 0] * many
        want = good[1].clone()
        want[[0, 1, 5]] = -1
        assert torch.equal(got[1], want.repeat(many))


def test_verify_takes_the_first_of_equal_logits():
    logits = torch.zeros(3, 2, 30000, device="cuda")
    logits[1, :, 20000:] = 1.0
    logits[2, 0, 29999] = 3.0
    drafts = torch.tensor([[0], [20000], [5]], device="cuda")
    u = torch.full((3, 1), 0.99, device="cuda")
    got = ethos_amd.verify_drafts(logits, drafts, u, u[:, 0].contiguous(), temperature=0.0)
    assert got[0].tolist() == [1, 1, 0] and got[1].tolist() == [0, 20000, 29999]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("mask", [-1e4, -1e9, -1e19, -1e20, -1e25, -1e30, "lowest"])
@pytest.mark.parametrize("b,m", [(5, 2), (130, 2)])
def test_verify_under_finite_masks(b, m, mask, dt):
    """Whole chunks (of 2,048 words, and of 8,192 where there are many rows) at one large finite value, and rows with nothing else."""
    V, T = 30001, DT[dt]
    value = torch.finfo(T).min if mask == "lowest" else mask
    logits, _, ua, us, _ = _verify_case(b, m, V, dt, "none", seed=11)
    logits[:, :, 2048:4096] = value
    logits[:, :, 8192:24576] = value
    logits[3] = value
    logits[4, :, 5000:] = value
    p = torch.softmax(logits[:, :m].float(), -1)
    drafts = torch.multinomial(p.view(-1, V), 1, generator=_gen(12)).view(b, m)
    drafts[0, 1] = 3000  # one of no weight
    for temperature in (1.0, 0.92, 1.03, 1.21, 0.7, 1e-6, 1e6, 0.0) if b == 5 else (1.0, 1.21, 0.0):
        for probs in (p, None):
            got = ethos_amd.verify_drafts(logits, drafts, ua, us, draft_probs=probs, temperature=temperature)
            assert (got[0].tolist(), got[1].tolist()) == _verify_oracle(logits, drafts, ua, us, probs, None, temperature), temperature


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("top", [1e16, -1e16, 1e20, -1e20, 1e30, -1e30, "highest", "lowest"])
def test_verify_of_rows_far_from_zero(top, dt):
    """Rows whose largest logits, some of each row's, are alike and far from zero: those share the weight, whatever the temperature."""
    b, m, V, T, g = 6, 3, 20001, DT[dt], _gen(13)
    top = torch.finfo(T).max if top == "highest" else torch.finfo(T).min if top == "lowest" else top
    high = torch.tensor(top, dtype=T, device="cuda")
    low = high.double() - abs(high.double()) / 64
    low = torch.tensor(max(float(low), float(torch.finfo(T).min)), dtype=T, device="cuda")
    logits = torch.where(torch.rand(b, m + 1, V, generator=g, device="cuda") < 0.3, high, low)
    drafts = logits[:, :m].float().argmax(-1)
    # draft probabilities around the model's: the random numbers accept some and refuse others
    count = (logits[:, :m] == logits[:, :m].amax(-1, keepdim=True)).sum(-1, keepdim=True)
    p = (logits[:, :m] == logits[:, :m].amax(-1, keepdim=True)).float() / count * (0.5 + torch.rand(b, m, V, generator=g, device="cuda") * 2)
    ua, us = torch.rand(b, m, generator=g, device="cuda"), torch.rand(b, generator=g, device="cuda")
    for temperature in (1.0, 0.8, 0.7, 1.3, 0.0):
        for probs in (p, None):
            got = ethos_amd.verify_drafts(logits, drafts, ua, us, draft_probs=probs, temperature=temperature)
            assert (got[0].tolist(), got[1].tolist()) == _verify_oracle(logits, drafts, ua, us, probs, None, temperature), temperature


def test_verified_tokens_are_distributed_as_the_model_says():
    """100,000 sequences of one draft over 12 words: each word's frequency as first token within five standard deviations."""
    n, V, g = 100000, 12, _gen(3)
    z = torch.randn(1, 2, V, generator=g, device="cuda").expand(n, 2, V).contiguous()
    q = torch.softmax(torch.randn(1, 1, V, generator=g, device="cuda"), -1).expand(n, 1, V).contiguous()
    drafts = torch.multinomial(q[0, 0], n, replacement=True, generator=g).view(n, 1)
    accepted, tokens = ethos_amd.verify_drafts(z, drafts, torch.rand(n, 1, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda"),
                                               draft_probs=q)
    first = torch.where(accepted > 0, drafts[:, 0], tokens)
    p = torch.softmax(z[0, 0].double(), -1)
    freq = torch.bincount(first, minlength=V).double() / n
    assert bool(((freq - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all())


def test_verify_of_more_sequences_than_a_launch_has_threads_for():
    """2^24 sequences and some, a draft for each but a few: over every launch's border, against float64."""
    n, V, g = (1 << 24) + 5, 8, _gen(8)
    for m in (0, 1):
        b = n if m == 0 else n // 2 + 1
        logits = (torch.randn(b, m + 1, V, generator=g, device="cuda") * 2).to(torch.bfloat16)
        drafts = torch.randint(0, V, (b, m), generator=g, device="cuda")
        ua, us = torch.rand(b, m, generator=g, device="cuda"), torch.rand(b, generator=g, device="cuda")
        accepted, tokens = ethos_amd.verify_drafts(logits, drafts, ua, us)
        z = logits.double()
        e = (z - z.amax(-1, keepdim=True)).exp()
        p = e / e.sum(-1, keepdim=True)
        del z, e
        took = torch.zeros(b, dtype=torch.int64, device="cuda")
        if m:
            took = (ua[:, 0].double() < p[:, 0].gather(1, drafts)[:, 0]).long()
        left = p.gather(1, took[:, None, None].expand(b, 1, V))[:, 0]
        if m:
            left.scatter_(1, drafts, torch.where(took[:, None] > 0, left.gather(1, drafts), 0.0))
        up = left.cumsum(1)
        del p, left
        above = us.double()[:, None] * up[:, -1:]
        want = (up <= above).sum(1)
        # (where a sum is within float64's rounding of the random number's place, either word is right)
        sure = ~((up - above).abs() < 1e-12).any(1)
        assert torch.equal(accepted.long(), took) and torch.equal(tokens[sure], want[sure]) and int((~sure).sum()) < 100
        if m == 0:
            greedy = ethos_amd.verify_drafts(logits, drafts, ua, us, temperature=0.0)[1]
            assert torch.equal(greedy, (logits[:, 0] == logits[:, 0].amax(-1, keepdim=True)).int().argmax(-1))


def test_verify_in_graphs_and_streams():
    cases = [_verify_case(9, 4, 30011, "bf16", "fp32", seed=s) for s in (4, 5)]
    want = [ethos_amd.verify_drafts(lo, d, ua, us, draft_probs=p) for lo, d, ua, us, p in cases]
    st = [t.clone() for t in cases[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ethos_amd.verify_drafts(st[0], st[1], st[2], st[3], draft_probs=st[4])
    for k in range(5):
        for s, t in zip(st, cases[k % 2]):
            s.copy_(t)
        graph.replay()
        eager = ethos_amd.verify_drafts(*cases[k % 2][:4], draft_probs=cases[k % 2][4])
        torch.cuda.synchronize()
        for a, b, c in zip(out, eager, want[k % 2]):
            assert torch.equal(a, c) and torch.equal(b, c)
    torch.cuda.synchronize()
    got = []
    for c in cases:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append([ethos_amd.verify_drafts(*c[:4], draft_probs=c[4]) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for xs, w in zip(got, want) for r in xs for x, y in zip(r, w))


# ------------------------------------------------------------------------------- refusals
def test_refusals():
    c = _case([9, 4], [2, 1], 4, 32, 16, 16, 16, 4, "fp32")

    def attend(**kw):
        d = dict(c, **kw)
        return ethos_amd.paged_attention(d["q"], d["w"], d["pool"], d["table"], d["lens"], d["starts"], d["rates"], d["scale"], d.get("out"))

    attend()
    with pytest.raises(RuntimeError, match="no gradient"):
        attend(q=c["q"].clone().requires_grad_())
    with torch.no_grad():
        attend(q=c["q"].clone().requires_grad_())
    with pytest.raises(RuntimeError, match="HIP device"):
        attend(lens=c["lens"].cpu())
    for bad in (dict(q=c["q"].bfloat16()), dict(w=c["w"].bfloat16())):
        with pytest.raises(TypeError):
            attend(**bad)
    for bad in (dict(q=c["q"].half()), dict(lens=c["lens"].long()), dict(starts=c["starts"].long()), dict(rates=c["rates"].double())):
        with pytest.raises((TypeError, RuntimeError)):
            attend(**bad)
    for bad in (dict(q=c["q"][0]), dict(q=c["q"][:, :3]), dict(w=c["w"][:-1]), dict(table=c["table"][:1]), dict(table=c["table"].long()),
                dict(table=c["table"].t().contiguous().t()), dict(starts=c["starts"][:-1]), dict(rates=c["rates"][:-1]), dict(pool=c["pool"][0]),
                dict(pool=c["pool"].transpose(0, 1)), dict(out=torch.empty(3, 63, device="cuda")), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=math.nan), dict(scale=math.inf), dict(pool=c["pool"][:, :3].contiguous())):
        with pytest.raises((RuntimeError, TypeError)):
            attend(**bad)
    rows, gain = torch.randn(3, 48, device="cuda"), torch.ones(32, device="cuda")
    a = (rows, gain, c["pool"], c["table"], c["lens"], c["starts"], c["rates"])
    ethos_amd.latent_append(*a)
    with pytest.raises(RuntimeError, match="no gradient"):
        ethos_amd.latent_append(rows, gain.clone().requires_grad_(), *a[2:])
    for i, bad in ((0, rows[:, :40]), (0, rows.bfloat16()), (1, gain[:30]), (1, torch.ones(64, device="cuda")), (2, c["pool"][0]),
                   (5, c["starts"][:2]), (6, c["rates"][:3])):
        with pytest.raises((RuntimeError, TypeError)):
            ethos_amd.latent_append(*a[:i], bad, *a[i + 1:])
    pool = torch.zeros(2, 5, 4, 8, device="cuda")
    for src, dst, error in (([0], [5], IndexError), ([-1], [2], IndexError), ([0, 1], [2, 2], ValueError), ([0, 1], [1, 2], ValueError),
                            ([0], [0], ValueError), ([0, 1], [2], ValueError), ([0.5], [1], TypeError),
                            (torch.tensor([0], device="cuda"), [1], TypeError), ([2 ** 40], [1], OverflowError), ([0, 5], [1, 2], IndexError)):
        with pytest.raises(error):
            ethos_amd.copy_pages(pool, src, dst)
    for bad in (pool.transpose(0, 1), pool[0, 0], pool.double(), pool.cpu()):
        with pytest.raises(RuntimeError):
            ethos_amd.copy_pages(bad, [0], [1])
    assert float(pool.abs().sum()) == 0.0
    logits, drafts, ua, us, p = _verify_case(3, 2, 50, "fp32", "fp32", seed=1)
    ok = dict(draft_probs=p, counts=i32([1, 2, 0]))
    ethos_amd.verify_drafts(logits, drafts, ua, us, **ok)
    for bad in ((logits.half(), drafts, ua, us, ok), (logits, drafts.int(), ua, us, ok), (logits, drafts, ua.double(), us, ok),
                (logits, drafts, ua, us, dict(draft_probs=p.half())), (logits, drafts, ua, us, dict(counts=torch.ones(3, device="cuda")))):
        with pytest.raises(TypeError):
            ethos_amd.verify_drafts(*bad[:4], **bad[4])
    for bad in ((logits[0], drafts, ua, us, {}), (logits, drafts[:, :1], ua, us, {}), (logits, drafts, ua[:2], us, {}),
                (logits, drafts, ua, us[:1], {}), (logits, drafts, ua, us, dict(draft_probs=p[:, :1])),
                (logits, drafts, ua, us, dict(counts=i32([1]))), (logits, drafts, ua, us, dict(temperature=-1.0)),
                (logits, drafts, ua, us, dict(temperature=1e-9)), (logits, drafts, ua, us, dict(temperature=math.nan)),
                (logits.cpu(), drafts, ua, us, {}), (logits.clone().requires_grad_(), drafts, ua, us, {})):
        with pytest.raises(RuntimeError):
            ethos_amd.verify_drafts(*bad[:4], **bad[4])
    assert isinstance(hip.FLOATS, tuple)
