"""The operators of a training step (ethos_amd.training) against float64.  Tolerances count
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


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------------------- cross entropy
def _ce_inputs(n, d, V, dt, seed=0, ignored=0.0):
    g = _gen(seed)
    w = torch.randn(V, d, generator=g, device="cuda") * 0.1
    labels = torch.randint(0, V, (n,), generator=g, device="cuda")
    h = torch.randn(n, d, generator=g, device="cuda") + w[labels] * 8.0
    if ignored >= 1.0:
        labels.fill_(-100)
    elif ignored > 0.0:
        labels[torch.rand(n, generator=g, device="cuda") < ignored] = -100
    return h.to(dt), w.to(dt), labels


def _ce_oracle(h, w, labels, reduction, gy):
    """(loss, dh, dw) in float64 and bounds of their errors: a logit's sum of d products is off by at
    most (d + 2) U times the sum of the products' sizes, the log-sum by that of its largest logit and a
    few roundings of its own; dl is off by its factor's error and (bf16) its rounding, the products
    with it by their sums of float32 additions, the results by their rounding.  (Kept exponentials,
    in bf16 alone: a step of 2^-11 more, or 2^-25 of the largest of their row.)"""
    x, m = h.double(), w.double()
    n, V, d = len(x), len(m), x.shape[1]
    keep = labels != -100
    at = torch.where(keep, labels, torch.zeros_like(labels))
    logits = x @ m.T
    e_logit = (d + 2) * U * (x.abs() @ m.abs().T).amax(1) if n else x.sum(1)
    lse = torch.logsumexp(logits, 1)
    e_lse = e_logit + 2.0 ** -20 + 8 * U * lse.abs() + (V.bit_length() + 8) * 2 * U
    zero = torch.zeros_like(lse)
    rows = torch.where(keep, lse - logits.gather(1, at[:, None])[:, 0], zero)
    e_rows = torch.where(keep, e_logit + e_lse + 2 * U * rows.abs(), zero)
    count = int(keep.sum())
    if reduction == "none":
        loss, e_loss = rows, e_rows
        g = gy.double()
    else:
        k = count if reduction == "mean" else 1
        loss, e_loss = rows.sum() / k, e_rows.sum() / k + 2 * U * rows.sum().abs() / k
        g = (gy.double() / k).expand(n) if k else zero
    g = torch.where(keep, g, zero)
    dl = (logits - lse[:, None]).exp()
    e_dl = dl * (e_logit + e_lse + 2.0 ** -20)[:, None]
    if h.dtype == torch.bfloat16:
        e_dl += dl * 2.0 ** -11 + dl.amax(1, keepdim=True) * 2.0 ** -25
    dl[torch.arange(n, device=x.device), at] -= 1.0
    # the label's value comes from the loss: an error of the loss moves it by as much
    e_dl[torch.arange(n, device=x.device), at] += e_rows + 4 * U
    t = half_step(h.dtype)
    dl *= g[:, None]
    e_dl = e_dl * g.abs()[:, None] + dl.abs() * (8 * U + (t if h.dtype == torch.bfloat16 else 0.0))
    dh, dw = dl @ m, dl.T @ x
    e_dh = e_dl @ m.abs() + (V + 64) * U * (dl.abs() @ m.abs()) + t * dh.abs() * 1.01
    e_dw = e_dl.T @ x.abs() + (n + 64) * U * (dl.abs().T @ x.abs()) + t * dw.abs() * 1.01
    return (loss, dh, dw), (e_loss, e_dh, e_dw)


def _within(got, want, bound, what):
    d = (got.double() - want).abs()
    bad = ~(d <= bound + 1e-30)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((d / (bound + 1e-30)).max()):.3g} bounds"


CE_SIZES = [(1, 64, 500), (2, 8, 1), (7, 1024, 1000), (255, 72, 511), (256, 64, 256), (257, 128, 513), (300, 1024, 3001),
            (1000, 200, 2000), (70, 40, 20011)]


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("n,d,V", CE_SIZES)
def test_cross_entropy_against_float64(n, d, V, dt, reduction):
    for ignored, keep in ((0.0, 1 << 30), (0.6, 1 << 30), (0.6, 0), (1.0, 1 << 30), (1.0, 0)):
        h, w, labels = _ce_inputs(n, d, V, DT[dt], seed=n + V, ignored=ignored)
        gy = torch.randn(n if reduction == "none" else (), generator=_gen(5), device="cuda")
        want, bound = _ce_oracle(h, w, labels, reduction, gy)
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction=reduction, keep_bytes=keep)
        assert loss.dtype == torch.float32
        dh, dw = torch.autograd.grad(loss, (a, b), gy)
        assert dh.dtype == h.dtype and dw.dtype == w.dtype and dh.shape == h.shape and dw.shape == w.shape
        with torch.no_grad():
            same = ethos_amd.linear_cross_entropy(h, w, labels, reduction=reduction)
        assert torch.equal(same.nan_to_num(7.0), loss.detach().nan_to_num(7.0))
        if not bool((labels != -100).any()):
            assert reduction != "mean" or bool(loss.isnan())
            assert reduction == "mean" or float(loss.detach().abs().sum()) == 0.0
            assert float(dh.float().abs().sum()) == 0.0 and float(dw.float().abs().sum()) == 0.0
            continue
        for got, x, e, what in zip((loss.detach(), dh, dw), want, bound, ("loss", "dh", "dw")):
            _within(got, x, e, f"{what} ignored={ignored}")
        assert bool((dh[labels == -100] == 0).all())
        loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction=reduction, keep_bytes=keep)
        again = torch.autograd.grad(loss, (a, b), gy, retain_graph=True)
        assert torch.equal(again[0], dh) and torch.equal(again[1], dw)
        # a retained graph's second backward, of another gradient: what the first was given has no part in it
        for got, x, e, what in zip(torch.autograd.grad(loss, (a, b), gy * 2.0), want[1:], bound[1:], ("dh", "dw")):
            _within(got * 0.5, x, e, f"second {what} ignored={ignored}")


@pytest.mark.parametrize("dt,n,d,V", [("bf16", 4096, 64, 140011), ("fp32", 2048, 64, 140011)])
def test_cross_entropy_several_pieces_of_vocabulary(dt, n, d, V):
    h, w, labels = _ce_inputs(n, d, V, DT[dt], seed=3, ignored=0.1)
    gy = torch.ones((), device="cuda")
    want, bound = _ce_oracle(h, w, labels, "mean", gy)  # 1.15 GB and 1.7 GB are not kept
    a, b = h.requires_grad_(), w.requires_grad_()
    loss = ethos_amd.linear_cross_entropy(a, b, labels)
    for got, x, e, what in zip((loss.detach(), *torch.autograd.grad(loss, (a, b), gy)), want, bound, ("loss", "dh", "dw")):
        _within(got, x, e, what)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("n,ignored,keep", [(700, 0.0, 1 << 30), (1300, 0.5, 0), (1300, 0.5, 1 << 30)])
def test_cross_entropy_in_the_largest_tiles(dt, n, ignored, keep):
    d, V = 264, 30011
    h, w, labels = _ce_inputs(n, d, V, DT[dt], seed=n, ignored=ignored)
    gy = torch.rand(n, generator=_gen(2), device="cuda")
    want, bound = _ce_oracle(h, w, labels, "none", gy)
    a, b = h.requires_grad_(), w.requires_grad_()
    loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction="none", keep_bytes=keep)
    for got, x, e, what in zip((loss.detach(), *torch.autograd.grad(loss, (a, b), gy)), want, bound, ("loss", "dh", "dw")):
        _within(got, x, e, what)


@pytest.mark.parametrize("n,d,ignored", [(2048, 264, 0.0), (2048, 40, 0.0), (2300, 320, 0.2)])
def test_cross_entropy_float32_passes_over_planes_in_the_largest_tiles(n, d, ignored):
    # 118 x 8 and x 9 tiles of 256, above three a CU: the planes' pairs in passes over one, five and (partly) five steps of 64
    h, w, labels = _ce_inputs(n, d, 30011, torch.float32, seed=d, ignored=ignored)
    gy = torch.rand(n, generator=_gen(2), device="cuda")
    want, bound = _ce_oracle(h, w, labels, "none", gy)
    a, b = h.requires_grad_(), w.requires_grad_()
    loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction="none")
    for got, x, e, what in zip((loss.detach(), *torch.autograd.grad(loss, (a, b), gy)), want, bound, ("loss", "dh", "dw")):
        _within(got, x, e, what)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("n,d,V", [(40, 136, 300), (130, 320, 260), (200, 384, 700), (330, 448, 129)])
def test_cross_entropy_of_a_few_steps(n, d, V, dt):
    # 3, 5, 6 and 7 steps of d; 1 to 6 of rows; 1 to 11 of words
    h, w, labels = _ce_inputs(n, d, V, DT[dt], seed=d)
    gy = torch.ones((), device="cuda")
    want, bound = _ce_oracle(h, w, labels, "sum", gy)
    a, b = h.requires_grad_(), w.requires_grad_()
    for keep in (0, 1 << 30):
        loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction="sum", keep_bytes=keep)
        for got, x, e, what in zip((loss.detach(), *torch.autograd.grad(loss, (a, b), gy)), want, bound, ("loss", "dh", "dw")):
            _within(got, x, e, what)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("keep", [0, 1 << 30])
def test_cross_entropy_of_equal_weights_rounds_rows_apart(reduction, keep):
    # every row's g lies in the middle of two bf16 values, and every label's probability is near 0: a rounding of g
    # itself would move both gradients by 2^-8.  Left: the results' rounding, at most 2^-8 / sqrt(3) on the root mean
    # square, and dl's, of 1 - p to 1, at most 2^-9.
    n, d, V = 512, 128, 3000
    g = _gen(23)
    h, w = torch.randn(n, d, generator=g, device="cuda").bfloat16() * 0.01, torch.randn(V, d, generator=g, device="cuda").bfloat16()
    labels = torch.randint(0, V, (n,), generator=g, device="cuda")
    gy = torch.full((n,) if reduction == "none" else (), 1.0 + 2.0 ** -8, device="cuda")
    (_, *want), _ = _ce_oracle(h, w, labels, reduction, gy)
    a, b = h.requires_grad_(), w.requires_grad_()
    loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction=reduction, keep_bytes=keep)
    for got, x, what in zip(torch.autograd.grad(loss, (a, b), gy), want, ("dh", "dw")):
        err = float((got.double() - x).norm() / x.norm())
        assert err <= math.hypot(2.0 ** -8 / math.sqrt(3.0), 2.0 ** -9), f"{what} {err}"


def test_cross_entropy_gradient_against_differences():
    h, w, labels = _ce_inputs(9, 16, 37, torch.float32, seed=2, ignored=0.3)
    labels[0] = 5
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    dh, dw = torch.autograd.grad(ethos_amd.linear_cross_entropy(a, b, labels), (a, b))
    f = lambda x, y: float(torch.nn.functional.cross_entropy(x.double() @ y.double().T, labels))  # noqa: E731
    g = _gen(1)
    for _ in range(4):
        u, v = torch.randn(h.shape, generator=g, device="cuda").double(), torch.randn(w.shape, generator=g, device="cuda").double()
        s = 1e-4
        diff = (f(h.double() + s * u, w.double() + s * v) - f(h.double() - s * u, w.double() - s * v)) / (2 * s)
        # central differences: s^2 / 6 of the third derivative, here below 1e-5 of the gradient's size
        mine = float((dh.double() * u).sum() + (dw.double() * v).sum())
        assert abs(mine - diff) <= 1e-5 * (float(dh.norm()) * float(u.norm()) + float(dw.norm()) * float(v.norm()))


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_cross_entropy_strides_shapes_and_one_gradient(dt):
    h, w, labels = _ce_inputs(60, 64, 300, DT[dt], seed=8)
    big = torch.zeros(60, 200, dtype=h.dtype, device="cuda")
    off = torch.zeros(60 * 64 + 1, dtype=h.dtype, device="cuda")
    views = [big[:, 8:72], off[1:].view(60, 64), h.t().contiguous().t(), big[:, 3:67]]
    want = ethos_amd.linear_cross_entropy(h, w, labels, reduction="none")
    for v in views:
        v.copy_(h)
        assert torch.equal(ethos_amd.linear_cross_entropy(v, w, labels, reduction="none"), want)
    three = ethos_amd.linear_cross_entropy(h.view(3, 20, 64), w, labels.view(3, 20), reduction="none")
    assert torch.equal(three, want.view(3, 20))
    moved = torch.zeros(300 * 64 + 1, dtype=w.dtype, device="cuda")[1:].view(300, 64).copy_(w)
    a, b, c = h.clone().requires_grad_(), w.clone().requires_grad_(), moved.requires_grad_()
    both = torch.autograd.grad(ethos_amd.linear_cross_entropy(a, b, labels), (a, b))
    assert torch.equal(torch.autograd.grad(ethos_amd.linear_cross_entropy(a, w, labels), a)[0], both[0])
    assert torch.equal(torch.autograd.grad(ethos_amd.linear_cross_entropy(h, b, labels), b)[0], both[1])
    assert torch.equal(torch.autograd.grad(ethos_amd.linear_cross_entropy(h, c, labels), c)[0], both[1])
    other = torch.where(labels % 3 == 0, torch.full_like(labels, 7), labels)
    mine = ethos_amd.linear_cross_entropy(h, w, other, ignore_index=7, reduction="none")
    assert torch.equal(mine, torch.where(other == 7, torch.zeros_like(want), want))


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_cross_entropy_masked_words_large_logits_and_wrong_labels(dt):
    h, w, labels = _ce_inputs(50, 64, 700, DT[dt], seed=4)
    h[:, 0] = 1.0
    w[300:600, 0] = -math.inf  # words that cannot be chosen, whole tiles among them
    labels.fill_(10)
    got = ethos_amd.linear_cross_entropy(h, w, labels, reduction="none")
    part = torch.cat([w[:300], w[600:]])
    want, bound = _ce_oracle(h, part, labels, "none", torch.ones(50, device="cuda"))
    _within(got, want[0], bound[0], "masked words")
    w[300:600, 0] = torch.finfo(w.dtype).min  # the lowest value, as masks often have it
    _within(ethos_amd.linear_cross_entropy(h, w, labels, reduction="none"), want[0], bound[0], "lowest values")
    # logits in the hundreds, of either sign
    h, w, labels = _ce_inputs(50, 64, 700, DT[dt], seed=5)
    a, b = (h * 40).requires_grad_(), w.requires_grad_()
    want, bound = _ce_oracle(a.detach(), b.detach(), labels, "sum", torch.ones((), device="cuda"))
    loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction="sum")
    for x, y, e, what in zip((loss.detach(), *torch.autograd.grad(loss, (a, b))), want, bound, ("loss", "dh", "dw")):
        _within(x, y, e, what)
    # a label outside the vocabulary, and a NaN in one row
    labels[3], labels[4] = 700, -1
    rows = ethos_amd.linear_cross_entropy(a, b, labels, reduction="none")
    assert rows.isnan().nonzero()[:, 0].tolist() == [3, 4]
    dh = torch.autograd.grad(rows, a, torch.ones(50, device="cuda"))[0]
    assert dh.isnan().any(1).nonzero()[:, 0].tolist() == [3, 4]
    h[9, 5] = math.nan
    labels[3], labels[4] = 1, 2
    assert ethos_amd.linear_cross_entropy(h, w.detach(), labels, reduction="none").isnan().nonzero()[:, 0].tolist() == [9]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_cross_entropy_with_labels_far_below(dt):
    """Rows of 300 whose labels' logits are 59, 61 and 400 below their sums."""
    h, w, labels = _ce_inputs(300, 64, 900, DT[dt], seed=12)
    g = _gen(4)
    for rows in ((5,), (5, 6, 7)):
        x = h.clone()
        for row, below in zip(rows, (59.0, 61.0, 400.0)):
            # a row against its label's: h = -c w, with c so that its logit is `below` under the others' sum
            v = w[labels[row]].double()
            c = below / float(v @ v)
            x[row] = (-c * v).to(x.dtype)
        a, b = x.requires_grad_(), w.clone().requires_grad_()
        gy = torch.rand(300, generator=g, device="cuda")
        want, bound = _ce_oracle(a.detach(), b.detach(), labels, "none", gy)
        loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction="none")
        for got, y, e, what in zip((loss.detach(), *torch.autograd.grad(loss, (a, b), gy)), want, bound, ("loss", "dh", "dw")):
            _within(got, y, e, f"{what} {rows}")


@pytest.mark.parametrize("mask", [-1e4, -1e6, -1e9, -1e10, -1e20, -1e30, -1e37])
@pytest.mark.parametrize("dt,n,V", [("bf16", 50, 700), ("fp32", 50, 700), ("bf16", 700, 30011), ("fp32", 2048, 30011)])
def test_cross_entropy_blocks_of_masked_words(dt, n, V, mask):
    """Words masked by a finite low logit, blocks of 64 and 128 of them in a row (in tiles of 128 and of 256): they
    have no part in the loss and no gradient, whichever way the backward goes."""
    h, w, labels = _ce_inputs(n, 64, V, DT[dt], seed=V)
    lo, hi = V // 3, 2 * V // 3
    h[:, 0] = 1.0
    w[lo:hi, 0] = mask
    labels %= lo
    gy = torch.rand(n, generator=_gen(7), device="cuda")
    want, bound = _ce_oracle(h, torch.cat([w[:lo], w[hi:]]), labels, "none", gy)
    for keep in (0, 1 << 30):
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction="none", keep_bytes=keep)
        dh, dw = torch.autograd.grad(loss, (a, b), gy)
        assert bool((dw[lo:hi] == 0).all()), f"masked words keep={keep}"
        for got, x, e, what in zip((loss.detach(), dh, torch.cat([dw[:lo], dw[hi:]])), want, bound, ("loss", "dh", "dw")):
            _within(got, x, e, f"{what} keep={keep}")


@pytest.mark.parametrize("size", [2 ** 9, -2 ** 9, 2 ** 12, -2 ** 12, 2 ** 20, 7 * 2 ** 31, -7 * 2 ** 31, 9 * 2 ** 31, -9 * 2 ** 31])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_cross_entropy_of_large_logits(dt, size):
    """Logits `size` plus small whole numbers (none above 2^20), exact in every partial sum.  Left are the roundings of
    the log-sum and of values scaled by log2(e), U |lse| each: they move the loss, and a probability by their exponential."""
    n, d, V = 40, 64, 700
    g = _gen(17)
    h = torch.randint(-1, 2, (n, d), generator=g, device="cuda").double()
    w = torch.randint(-1, 2, (V, d), generator=g, device="cuda").double()
    if abs(size) > 2 ** 20:
        w.zero_()
    h[:, 0], w[:, 0] = 1.0, float(size)
    labels = torch.randint(0, V, (n,), generator=g, device="cuda")
    x = h @ w.T
    lse = torch.logsumexp(x, 1)
    at = torch.arange(n, device="cuda"), labels
    rows = lse - x[at]
    e_loss = 2 * U * lse.abs() + 2.0 ** -18 + 2 * U * rows
    dl = (x - lse[:, None]).exp()
    e_dl = dl * torch.expm1(3 * U * lse.abs() + 2.0 ** -17).clamp(max=1e30)[:, None] + dl * 2.0 ** -11 + 2.0 ** -25
    dl[at] -= 1.0
    t = half_step(DT[dt])
    e_dl += dl.abs() * (8 * U + (t if dt == "bf16" else 0.0))
    dh, dw = (dl @ w)[:, 1:], dl.T @ h
    e_dh = (e_dl @ w.abs() + (V + 64) * U * (dl.abs() @ w.abs()))[:, 1:] + t * dh.abs() * 1.01
    e_dw = e_dl.T @ h.abs() + (n + 64) * U * (dl.abs().T @ h.abs()) + t * dw.abs() * 1.01
    for keep in (0, 1 << 30):
        a, b = h.to(DT[dt]).requires_grad_(), w.to(DT[dt]).requires_grad_()
        loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction="none", keep_bytes=keep)
        got = torch.autograd.grad(loss, (a, b), torch.ones(n, device="cuda"))
        _within(loss.detach(), rows, e_loss, f"loss keep={keep}")
        _within(got[0][:, 1:], dh, e_dh, f"dh keep={keep}")
        _within(got[1], dw, e_dw, f"dw keep={keep}")


@pytest.mark.parametrize("keep", [0, 1 << 30])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_cross_entropy_of_a_row_without_any_word(dt, keep):
    # every logit of row 3 is -inf, so none of its probabilities is a number
    h, w, labels = _ce_inputs(20, 64, 700, DT[dt], seed=9)
    h[:, 0], w[:, 0] = 1.0, 0.25
    h[3, 0] = -math.inf
    a, b = h.requires_grad_(), w.requires_grad_()
    loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction="none", keep_bytes=keep)
    assert loss.isnan().nonzero()[:, 0].tolist() == [3]
    dh, dw = torch.autograd.grad(loss, (a, b), torch.ones(20, device="cuda"))
    assert dh.isnan().all(1).nonzero()[:, 0].tolist() == [3] and not bool(dh[:3].isnan().any() | dh[4:].isnan().any())
    assert bool(dw.isnan().all())


@pytest.mark.parametrize("keep", [0, 1 << 30])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_cross_entropy_is_never_negative(dt, keep):
    """Rows along their labels' rows: the labels' logits (some 5,000) are all of their log-sums but e^-4000, so a loss is the
    difference of two roundings of one sum of d products.  It is not negative, and its gradient moves no logit of a label down."""
    n, d, V = 256, 1024, 512
    g = _gen(31)
    w = torch.randn(V, d, generator=g, device="cuda").to(DT[dt])
    labels = torch.randint(0, V, (n,), generator=g, device="cuda")
    h = w[labels] * 5.0
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction="none", keep_bytes=keep)
    dh, _ = torch.autograd.grad(loss, (a, b), torch.ones(n, device="cuda"))
    assert bool((loss >= 0).all()), float(loss.min())
    _within(loss.detach(), torch.zeros(n, device="cuda").double(), 2 * (d + 2) * U * (h.double().abs() * w[labels].double().abs()).sum(1), "loss")
    assert float((dh.double() * w[labels].double()).sum(1).max()) <= 0.0
    assert float(ethos_amd.linear_cross_entropy(h, w, labels)) >= 0.0


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cross_entropy_of_no_rows(dt, reduction):
    h, w = torch.zeros(2, 0, 16, device="cuda", dtype=DT[dt]), torch.randn(9, 16, device="cuda", generator=_gen(0)).to(DT[dt])
    w[0, 0], w[1, 1] = math.inf, math.nan
    labels = torch.zeros(2, 0, dtype=torch.int64, device="cuda")
    a, b = h.requires_grad_(), w.requires_grad_()
    loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction=reduction)
    assert loss.dtype == torch.float32 and loss.shape == ((2, 0) if reduction == "none" else ()) and loss.requires_grad
    value = loss.detach()
    assert reduction == "none" or (float(value) == 0.0 if reduction == "sum" else math.isnan(float(value)))
    # as for a batch of ignored positions
    dh, dw = torch.autograd.grad(loss, (a, b), torch.ones_like(loss))
    assert dh.shape == h.shape and dh.dtype == h.dtype and dw.dtype == w.dtype and bool((dw == 0).all()) and dw.shape == w.shape
    with torch.no_grad():
        same = ethos_amd.linear_cross_entropy(a, b, labels, reduction=reduction)
    assert not same.requires_grad and torch.equal(same.nan_to_num(7.0), loss.detach().nan_to_num(7.0))


def test_cross_entropy_table_past_32_bits():
    n, d, V = 5, 16384, 140000  # 4.6 GB
    w = torch.empty(V, d, dtype=torch.bfloat16, device="cuda")
    g = _gen(6)
    for part in w.split(10000):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * 0.02)
    labels = torch.tensor([0, V - 1, 131072, -100, 139000], device="cuda")
    h = torch.randn(n, d, generator=g, device="cuda").to(torch.bfloat16)
    logits = torch.cat([h.double() @ p.double().T for p in w.split(10000)], 1)
    size = torch.cat([h.double().abs() @ p.double().abs().T for p in w.split(10000)], 1).amax()
    a, b = h.requires_grad_(), w.requires_grad_()
    loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction="sum")
    keep = labels >= 0
    logp = torch.log_softmax(logits[keep], 1)
    want = -logp.gather(1, labels[keep][:, None]).sum()
    e = float((d + 2) * U * size)
    assert abs(float(loss.detach()) - float(want)) <= 4 * (2 * e + 2.0 ** -19 + 32 * U * 20)
    dh, dw = torch.autograd.grad(loss, (a, b))
    dl = logp.exp()
    dl[torch.arange(4, device="cuda"), labels[keep]] -= 1.0
    u = half_step(torch.bfloat16)
    for v in (0, 1, 65535, 65536, 131071, 131072, 131073, V - 2, V - 1):
        x = dl[:, v] @ h.detach()[keep].double()
        _within(dw[v], x, (u + 2.0 ** -11 + 3 * e + 2.0 ** -19) * (dl[:, v].abs() @ h.detach()[keep].double().abs()) + u * x.abs(), f"dw[{v}]")
    x = sum(dl[:, i:i + 10000] @ p.double() for i, p in zip(range(0, V, 10000), w.detach().split(10000)))
    m = sum(dl[:, i:i + 10000].abs() @ p.double().abs() for i, p in zip(range(0, V, 10000), w.detach().split(10000)))
    _within(dh[keep], x, (u + 2.0 ** -10 + 3 * e + 2.0 ** -19 + V * U) * m + u * x.abs(), "dh")


# ------------------------------------------------------------------------------- embedding
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("shape,V,d", [((1,), 5, 1), ((64,), 100277, 1024), ((3, 500), 5003, 101), ((8192,), 900, 72), ((2, 33), 40, 6),
                                       ((20000,), 30, 20), ((0,), 7, 8)])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_embedding_against_float64(shape, V, d, dt, itype):
    g = _gen(V + d)
    n = math.prod(shape)
    ids = (torch.rand(shape, generator=g, device="cuda") ** 3 * V).long().clamp_(max=V - 1)
    w = torch.randn(V, d, generator=g, device="cuda").to(DT[dt])
    for scale, padding in ((1.0, None), (27.7, 0), (0.5, -1)):
        p = w.clone().requires_grad_()
        y = ethos_amd.embedding(ids.to(itype), p, scale=scale, padding_idx=padding)
        assert torch.equal(y.detach(), (w[ids].float() * scale).to(w.dtype))
        dy = torch.randn(y.shape, generator=g, device="cuda").to(w.dtype)
        dw = torch.autograd.grad(y, p, dy)[0]
        x = dy.double().view(n, d)
        if padding is not None:
            x = x * (ids.view(-1) != padding % V)[:, None]
        want = torch.zeros(V, d, dtype=torch.float64, device="cuda").index_add_(0, ids.view(-1), x) * scale
        size = torch.zeros(V, d, dtype=torch.float64, device="cuda").index_add_(0, ids.view(-1), x.abs()) * scale
        uses = torch.bincount(ids.view(-1), minlength=V).double()[:, None]
        _within(dw, want, (uses + 4) * U * size + half_step(w.dtype) * want.abs() * 1.01, f"dw scale={scale} padding={padding}")
        assert torch.equal(torch.autograd.grad(ethos_amd.embedding(ids.to(itype), p, scale=scale, padding_idx=padding), p, dy)[0], dw)


def test_embedding_ids_outside_the_table_and_views():
    w = torch.randn(50, 24, device="cuda", generator=_gen(0)).to(torch.bfloat16)
    ids = torch.tensor([3, -1, 50, 49, 2 ** 40], device="cuda")
    p = w.clone().requires_grad_()
    y = ethos_amd.embedding(ids, p)
    assert y.isnan().all(1).tolist() == [False, True, True, False, True]
    dy = torch.ones(24, 5, device="cuda", dtype=torch.bfloat16).t()  # rows not contiguous
    dw = torch.autograd.grad(y, p, dy)[0]
    assert dw.float().sum(1).nonzero()[:, 0].tolist() == [3, 49]
    wide = torch.zeros(50, 48, device="cuda", dtype=torch.bfloat16)
    wide[:, 1:25] = w
    assert torch.equal(ethos_amd.embedding(ids[:1], wide[:, 1:25]), w[3:4])
    odd = torch.zeros(50 * 24 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(50, 24).copy_(w)
    assert torch.equal(ethos_amd.embedding(ids.view(-1)[::3], odd), w[[3, 49]])


def test_embedding_gradient_of_more_runs_than_a_launch_takes_at_once():
    # 2^24 + 2 runs of eight positions; whole numbers, whose sums stay below 2^24 and so are exact in float32
    n, V, d = 2 ** 27 + 13, 1000, 2
    g = _gen(29)
    ids = torch.randint(0, V, (n,), generator=g, device="cuda", dtype=torch.int32)
    ids[-9:] = V - 1
    p = torch.zeros(V, d, device="cuda", requires_grad=True)
    y = ethos_amd.embedding(ids, p)
    dy = torch.randint(-8, 9, (n, d), generator=g, device="cuda", dtype=torch.int8).float()
    dw = torch.autograd.grad(y, p, dy)[0]
    want = torch.zeros(V, d, dtype=torch.float64, device="cuda")
    for i, x in zip(ids.split(2 ** 24), dy.split(2 ** 24)):
        want.index_add_(0, i, x.double())
    assert float(want.abs().max()) < 2 ** 24 and torch.equal(dw.double(), want)


# ------------------------------------------------------------------------------- balance
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
@pytest.mark.parametrize("n,H,k,E", [(1, 1, 1, 1), (1, 2, 4, 256), (37, 3, 5, 1000), (500, 4, 8, 4096), (1000, 8, 16, 262144),
                                     (300, 4, 8, 600000)])
def test_balance_against_float64(n, H, k, E, dt, itype):
    g = _gen(n + E)
    gates = torch.softmax(torch.randn(n, H, k, generator=g, device="cuda"), -1).to(DT[dt]).requires_grad_()
    ids = (torch.rand(n, H, k, generator=g, device="cuda") ** 4 * E).long().clamp_(max=E - 1)
    loss, counts = ethos_amd.balance_loss(gates, ids.to(itype), E)
    want = torch.bincount(ids.flatten(), minlength=E)
    assert counts.dtype == torch.int32 and torch.equal(counts.long(), want) and not counts.requires_grad
    slope = want.double()[ids] * (E / (float(n) * H * k) / (float(n) * H))
    x = (slope * gates.detach().double()).sum()
    assert abs(float(loss.detach()) - float(x)) <= 2 * U * float(x)
    dg = torch.autograd.grad(loss * 0.5, gates)[0]
    _within(dg, slope * 0.5, (half_step(gates.dtype) + 2 * U) * 1.01 * slope * 0.5, "dgates")
    # gates that are not contiguous, in other leading shapes
    wide = torch.zeros(n, H, 2 * k, device="cuda", dtype=gates.dtype)
    wide[..., ::2] = gates.detach()
    l2, c2 = ethos_amd.balance_loss(wide[..., ::2][None], ids[None].to(itype), E)
    assert torch.equal(l2, loss.detach()) and torch.equal(c2, counts)


def test_balance_even_routing_ids_outside_and_no_tokens():
    ids = torch.arange(64, device="cuda", dtype=torch.int32).view(8, 2, 4)
    gates = torch.full((8, 2, 4), 0.25, device="cuda", requires_grad=True)
    loss, counts = ethos_amd.balance_loss(gates, ids, 64)
    assert float(loss.detach()) == 1.0 and bool((counts == 1).all())
    bad = ids.clone()
    bad[0, 0, :2] = torch.tensor([-1, 64], dtype=torch.int32, device="cuda")
    loss, counts = ethos_amd.balance_loss(gates, bad, 64)
    assert int(counts.sum()) == 62
    assert (torch.autograd.grad(loss, gates)[0] == 0).nonzero().tolist() == [[0, 0, 0], [0, 0, 1]]
    loss, counts = ethos_amd.balance_loss(gates[:0], ids[:0], 64)
    assert float(loss.detach()) == 0.0 and int(counts.sum()) == 0
    assert torch.autograd.grad(loss, gates)[0].abs().sum() == 0


# ------------------------------------------------------------------------------- clipping
def _norm(ts, norm):
    ts = [t.double().flatten() for t in ts if t.numel()]
    return torch.cat(ts).abs().max() if norm == math.inf else torch.cat(ts).norm()


@pytest.mark.parametrize("norm", [2.0, math.inf])
@pytest.mark.parametrize("share", [0.1, 2.0])
@pytest.mark.parametrize("in_place", [False, True])
def test_clip_against_float64(norm, share, in_place):
    g = _gen(11)
    shapes = [(1,), (300,), (0,), (33, 77), (70001,), ()] + [(i % 13 + 1, i % 7 + 1) for i in range(290)] + [(513, 257)]
    grads = [(torch.randn(s, generator=g, device="cuda") * 10.0 ** (i % 3)).to(torch.float32 if i % 5 == 0 else torch.bfloat16)
             for i, s in enumerate(shapes)]
    # a view at an odd address, and transposed memory
    grads += [torch.randn(1001, generator=g, device="cuda").bfloat16()[1:], torch.randn(40, 60, generator=g, device="cuda").t()]
    size = _norm(grads, norm)
    top = float(size) * share
    factor = min(1.0, top / (float(size) + 1e-6))
    want = [t.double() * factor for t in grads]
    if in_place:
        out, versions = grads, [t._version for t in grads]
    else:
        flat = torch.empty(sum(t.numel() for t in grads if t.dtype == torch.bfloat16) + 1, dtype=torch.bfloat16, device="cuda")[1:]
        parts = iter(flat.split([t.numel() for t in grads if t.dtype == torch.bfloat16]))
        out = [next(parts).view(t.shape) if t.dtype == torch.bfloat16 else torch.empty_like(t) for t in grads]
        keep = [t.clone() for t in grads]
    total = ethos_amd.clip_grads(grads, top, norm_type=norm, out=None if in_place else out)
    assert abs(float(total) - float(size)) <= 2 * U * float(size)
    for i, (o, x) in enumerate(zip(out, want)):
        # the factor's rounding, the product's and the result's
        _within(o, x, (half_step(o.dtype) + 3 * U) * 1.01 * x.abs(), f"tensor {i}")
    if in_place:
        assert all(t._version > v for t, v in zip(grads, versions))
    else:
        assert all(torch.equal(t, k) for t, k in zip(grads, keep))


@pytest.mark.parametrize("norm", [2.0, math.inf])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_clip_of_many_pieces(norm, dt):
    # one tensor of 2^27 + 10001 values and 1,200 of a few
    g = _gen(19)
    big = torch.randn(2 ** 27 + 10001, generator=g, device="cuda", dtype=DT[dt])
    big[-1] = 100.0
    grads = [big] + [t.clone() for t in torch.randn(1200, 3, generator=g, device="cuda").to(DT[dt])]
    size = float(_norm(grads, norm))
    keep = [t.clone() for t in grads]
    total = ethos_amd.clip_grads(grads, 0.5 * size, norm_type=norm)
    assert abs(float(total) - size) <= 2 * U * size
    factor = 0.5 * size / (size + 1e-6)
    for i, (o, k) in enumerate(zip(grads, keep)):
        x = k.double() * factor
        _within(o, x, (half_step(o.dtype) + 3 * U) * 1.01 * x.abs(), f"tensor {i}")


def test_clip_extreme_values():
    big = torch.full((100000,), 3e38, device="cuda")
    total = ethos_amd.clip_grads([big], 1.0)
    # the norm, 3e38 sqrt(1e5), is above float32; the factor is a subnormal of half step 2^-150
    assert math.isinf(float(total))
    want = 1e5 ** -0.5
    assert abs(float(big[0]) - want) <= want * (2.0 ** -150 * 3e38 / want + 4 * U) and bool((big == big[0]).all())
    big = torch.full((4,), 1e30, device="cuda")  # squares above float32, the norm within it
    assert abs(float(ethos_amd.clip_grads([big], 1.0)) / 2e30 - 1) <= 4 * U and abs(float(big[0]) - 0.5) <= 4 * U
    small = torch.full((4,), 1e-30, device="cuda", dtype=torch.bfloat16)
    v = float(small[0])
    assert abs(float(ethos_amd.clip_grads(small, 1.0)) / (2 * v) - 1) <= 4 * U and float(small[0]) == v
    for norm in (2.0, math.inf):
        ts = [torch.ones(50, device="cuda"), torch.ones(70000, device="cuda")]
        ts[1][66000] = math.nan
        assert math.isnan(float(ethos_amd.clip_grads(ts, 1.0, norm_type=norm))) and all(bool(t.isnan().all()) for t in ts)
    ts = torch.ones(9, device="cuda")
    assert float(ethos_amd.clip_grads(ts, 0.0)) == 3.0 and float(ts.abs().sum()) == 0.0
    assert float(ethos_amd.clip_grads([], 1.0)) == 0.0 and float(ethos_amd.clip_grads([torch.empty(0, device="cuda")], 1.0)) == 0.0


# ------------------------------------------------------------------------------- refusals
def test_refusals():
    h, w, l = torch.zeros(4, 16, device="cuda"), torch.zeros(9, 16, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    ce = ethos_amd.linear_cross_entropy
    for bad, kind in (((h, w, l.int()), TypeError), ((h.half(), w.half(), l), TypeError), ((h, w.bfloat16(), l), TypeError),
                      ((h[:, :8], w, l), RuntimeError), ((h[:, :12], w[:, :12], l), RuntimeError), ((h, w, l[:3]), RuntimeError),
                      ((h, w[:0], l), RuntimeError), ((h.cpu(), w, l), RuntimeError), ((h, w, l.cpu()), RuntimeError)):
        with pytest.raises(kind):
            ce(*bad)
    with pytest.raises(ValueError):
        ce(h, w, l, reduction="max")
    for bad, kw, kind in (((l, w.half()), {}, TypeError), ((l.float(), w), {}, TypeError), ((l, w[0]), {}, RuntimeError),
                          ((l, w), dict(padding_idx=9), ValueError), ((l.cpu(), w), {}, RuntimeError)):
        with pytest.raises(kind):
            ethos_amd.embedding(*bad, **kw)
    g, i = torch.zeros(4, 2, 3, device="cuda"), torch.zeros(4, 2, 3, dtype=torch.int32, device="cuda")
    for bad, kind in (((g.half(), i, 5), TypeError), ((g, i.float(), 5), TypeError), ((g, i[:3], 5), RuntimeError), ((g, i, 0), ValueError),
                      ((g[0, 0], i[0, 0], 5), RuntimeError), ((g, i.cpu(), 5), RuntimeError)):
        with pytest.raises(kind):
            ethos_amd.balance_loss(*bad)
    for bad, kw, kind in ((([h, w], 1.0), dict(norm_type=1), ValueError), (([h], -1.0), {}, ValueError), (([h], math.nan), {}, ValueError),
                          (([h, h], 1.0), {}, ValueError), (([h], 1.0), dict(out=[w]), RuntimeError), (([h], 1.0), dict(out=[]), ValueError),
                          (([h.half()], 1.0), {}, TypeError), (([h.cpu()], 1.0), {}, RuntimeError), (([None], 1.0), {}, TypeError)):
        with pytest.raises(kind):
            ethos_amd.clip_grads(*bad, **kw)


def test_a_weight_changed_before_the_backward_is_noticed():
    h, w, labels = _ce_inputs(8, 16, 30, torch.float32)
    w.requires_grad_()
    loss = ethos_amd.linear_cross_entropy(h, w, labels)
    with torch.no_grad():
        w.add_(1.0)
    with pytest.raises(RuntimeError):
        loss.backward()


# ------------------------------------------------------------------------------- streams and graphs
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_on_another_stream_and_in_a_graph(dt):
    """Forward and backward of all four in one captured graph, replayed on new inputs between the
    program's own eager work, against the eager results."""
    n, d, V, H, k, E = 130, 64, 700, 2, 4, 256
    w = (torch.randn(V, d, generator=_gen(0), device="cuda") * 0.1).to(DT[dt]).requires_grad_()
    ids, labels = torch.zeros(n, dtype=torch.int64, device="cuda"), torch.zeros(n, dtype=torch.int64, device="cuda")
    experts = torch.zeros(n, H, k, dtype=torch.int64, device="cuda")
    gates = torch.full((n, H, k), 0.25, device="cuda", dtype=DT[dt], requires_grad=True)

    def step():
        x = ethos_amd.embedding(ids, w, scale=2.0)
        loss = ethos_amd.linear_cross_entropy(x, w, labels)
        aux, counts = ethos_amd.balance_loss(gates, experts, E)
        grads = torch.autograd.grad(loss + 0.1 * aux, (w, gates))
        out = [torch.empty_like(t) for t in grads]
        total = ethos_amd.clip_grads(list(grads), 0.05, out=out)
        return [loss.detach(), aux.detach(), counts, total, *out]

    def inputs(seed):
        g = _gen(seed)
        ids.copy_(torch.randint(0, V, (n,), generator=g, device="cuda"))
        labels.copy_(torch.randint(0, V, (n,), generator=g, device="cuda"))
        labels[seed::3] = -100
        experts.copy_(torch.randint(0, E, (n, H, k), generator=g, device="cuda"))

    inputs(1)
    side = torch.cuda.Stream()
    want = step()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = [step() for _ in range(3)]
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (2, 3, 4, 5):
        inputs(seed)
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), seed


def test_a_backward_captured_alone_can_be_replayed():
    h, w, labels = _ce_inputs(130, 64, 700, torch.bfloat16, seed=3)
    a, b, gy = h.requires_grad_(), w.requires_grad_(), torch.ones((), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = ethos_amd.linear_cross_entropy(a, b, labels)
        want = torch.autograd.grad(ethos_amd.linear_cross_entropy(a, b, labels, keep_bytes=0), (a, b), gy)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = torch.autograd.grad(loss, (a, b), gy, retain_graph=True)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        # the eager graph's own backward still has what the forward left
        eager = torch.autograd.grad(loss, (a, b), gy)
        again = torch.autograd.grad(ethos_amd.linear_cross_entropy(a, b, labels), (a, b), gy)
        assert torch.equal(eager[0], again[0]) and torch.equal(eager[1], again[1])


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_a_backward_captured_apart_from_its_forward_can_be_replayed(dt):
    """Forward and backward in graphs of their own, as wrappers of callables capture them: the backward's replays after
    one replay of the forward, each of another gradient, against eager results."""
    h, w, labels = _ce_inputs(130, 64, 700, DT[dt], seed=3)
    a, b, gy = h.requires_grad_(), w.requires_grad_(), torch.ones(130, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def eager():
        return torch.autograd.grad(ethos_amd.linear_cross_entropy(a, b, labels, reduction="none", keep_bytes=0), (a, b), gy)

    with torch.cuda.stream(side):
        eager()
        torch.cuda.synchronize()
        forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(forward, stream=side):
            loss = ethos_amd.linear_cross_entropy(a, b, labels, reduction="none")
        with torch.cuda.graph(backward, stream=side):
            got = torch.autograd.grad(loss, (a, b), gy, retain_graph=True)
        for seed in (1, 2):
            labels.copy_(torch.randint(0, 700, (130,), generator=_gen(seed), device="cuda"))
            forward.replay()
            for scale in (1.0, -3.0, 0.5):
                gy.copy_(torch.rand(130, generator=_gen(seed), device="cuda") * scale)
                backward.replay()
                torch.cuda.synchronize()
                want = eager()
                torch.cuda.synchronize()
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (seed, scale)


@pytest.mark.parametrize("train", [False, True])
def test_no_copy_of_the_logits(train):
    """Without gradients, or with none of the exponentials kept, the loss's memory beside its inputs and
    outputs stays a small part of the logits'; what is kept for a backward is gone after it."""
    h, w, labels = _ce_inputs(4096, 64, 100000, torch.bfloat16)
    h.requires_grad_(train)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss = ethos_amd.linear_cross_entropy(h, w, labels, keep_bytes=0 if train else 1 << 30)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 4096 * 100000 * 4 / 20
    if train:
        del loss
        loss = ethos_amd.linear_cross_entropy(h, w, labels)
        assert torch.cuda.memory_allocated() - before > 4096 * 100000 * 2
        dh = torch.autograd.grad(loss, h)[0]
        assert torch.cuda.memory_allocated() - before < 4096 * 100000 * 2 / 20 and dh.shape == h.shape


def test_wrappers_refuse_other_devices(monkeypatch):
    monkeypatch.setattr(hip, "_current_device", lambda: 1)
    with pytest.raises(RuntimeError):
        ethos_amd.embedding(torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(4, 8, device="cuda"))


def test_wrappers_refuse_what_the_kernels_cannot_read():
    """Each wrapper with one argument wrong: on the host, of another type, of too few values."""
    z = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731
    i32, i64 = torch.int32, torch.int64

    def refused(call, good, **bad):
        call(**good)
        for name, values in bad.items():
            for v in values:
                with pytest.raises((RuntimeError, TypeError)):
                    call(**{**good, name: v})

    ce = dict(h=z(4, 16), w=z(9, 16), labels=z(4, dt=i64), ignore_index=-100, reduction="none")
    refused(hip.linear_ce, ce, h=(z(4, 16).cpu(), z(4, 16, dt=torch.bfloat16), z(3, 16), z(4, 8), z(16, 4).t(), z(2, 2, 16), None),
            w=(z(9, 16).cpu(), z(9, 8), z(16, 9).t()), labels=(z(4).long().cpu(), z(4, dt=i32), z(5, dt=i64)))
    _, state, _ = hip.linear_ce(**ce)
    grad = dict(state=state, exps=None, w=ce["w"], dloss=z(4), n=4, reduction="none", want_h=True, want_w=True)
    refused(hip.linear_ce_grad, grad, state=(state.cpu(), state[:1], state.int()), w=(ce["w"].cpu(), z(16, 9).t()),
            dloss=(z(4).cpu(), z(3), z(1), z(4).double(), z(8)[::2]), exps=(state.cpu(), state))
    keys = dict(keys=z(4, dt=i32), dy=z(4, 16), vocab=9, scale=1.0)
    refused(hip.embedding_grad, keys, keys=(z(4, dt=i64), z(4, dt=i32).cpu(), z(5, dt=i32)), dy=(z(4, 16).cpu(), z(3, 16), z(16, 4).t()))
    bal = dict(gates=z(4, 2, 3), ids=z(4, 2, 3, dt=i32), n_experts=5)
    refused(hip.balance, bal, gates=(z(3, 2, 3), z(4, 2, 3).cpu(), z(6)), ids=(z(4, 2, 2, dt=i32), z(4, 2, 3, dt=i32).cpu()))
    back = dict(ids=bal["ids"], counts=z(5, dt=i32), dloss=z(), dtype=torch.float32)
    refused(hip.balance_grad, back, ids=(bal["ids"].cpu(), z(4, dt=i32)), counts=(z(5, dt=i32).cpu(), z(5, dt=i64)),
            dloss=(z().cpu(), z().double(), z(2)))


# ------------------------------------------------------------------------------- the model's loss
def _tiny_model(seed=0):
    from ethos_amd.model import CompressedMoEModel
    from ethos_amd.workloads import make_lm_inputs

    cfg, sd, ids = make_lm_inputs(seed=seed)
    m = CompressedMoEModel(cfg)
    m.load_state_dict(sd)
    labels = torch.roll(ids, -1, 1)
    labels[:, -1] = -100
    return cfg, m.cuda().train(), ids.cuda(), labels.cuda()


def test_model_loss_against_torch_operations():
    """CompressedMoEModel.loss against torch's cross entropy of the logits: the blocks are the same
    computation, linear in the last rows' gradient, which the two form with sums of up to 500 + 64
    float32 terms: (500 + 64) U = 3.4e-5 of its size."""
    cfg, m, ids, labels = _tiny_model()
    parts = m.loss(ids, labels)
    assert parts.balance is None and parts.counts == [] and torch.equal(parts.loss.detach(), parts.cross_entropy)
    params = [p for p in m.parameters()]
    got = torch.autograd.grad(parts.loss, params)
    want = torch.nn.functional.cross_entropy(m(ids).view(-1, cfg.vocab_size), labels.view(-1), ignore_index=-100)
    assert abs(float(parts.cross_entropy) - float(want.detach())) <= (64 + 16) * U * 16
    ref = torch.autograd.grad(want, params)
    for (name, _), a, b in zip(m.named_parameters(), got, ref):
        assert float((a - b).norm()) <= 3.4e-5 * 3 * float(b.norm()) + 1e-12, name


def test_model_trains_with_balance_and_clipping():
    cfg, m, ids, labels = _tiny_model(1)
    experts = cfg.num_layers - cfg.num_dense_layers
    params = list(m.parameters())
    opt = torch.optim.SGD(params, lr=0.5)
    losses = []
    for step in range(12):
        parts = m.loss(ids, labels, balance_weight=0.01)
        assert len(parts.counts) == experts and all(int(c.sum()) == ids.numel() * cfg.top_k * cfg.num_routing_heads for c in parts.counts)
        assert abs(float(parts.loss.detach()) - float(parts.cross_entropy) - 0.01 * float(parts.balance)) <= 4 * U * float(parts.loss.detach())
        opt.zero_grad()
        parts.loss.backward()
        grads = [p.grad for p in params]
        before = float(_norm(grads, 2.0))
        total = ethos_amd.clip_grads(grads, 1.0)
        assert abs(float(total) - before) <= 2 * U * before and float(_norm(grads, 2.0)) <= 1.0 + 1e-5
        opt.step()
        losses.append(float(parts.cross_entropy))
    assert losses[-1] < 0.8 * losses[0]
    # the balance loss reaches the router: its gradient alone is not zero there
    parts = m.loss(ids, labels, balance_weight=1.0)
    plain = m.loss(ids, labels)
    key = m.layers[-1].mlp.router.sub_keys_1.weight
    a, b = torch.autograd.grad(parts.loss, key)[0], torch.autograd.grad(plain.loss, key)[0]
    assert float((a - b).norm()) > 0.0
    m.eval()
    with torch.no_grad():
        parts = m.loss(ids, labels, balance_weight=0.5)
        assert not parts.loss.requires_grad and len(parts.counts) == experts
