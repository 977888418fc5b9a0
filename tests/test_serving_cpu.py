"""The serving operators' refusals that need no GPU: argument errors of the C-ABI come back as codes
before anything is enqueued, and the Python entry points name what is wrong."""
import ctypes

import pytest
import torch

import ethos_amd
from ethos_amd import _lib, hip, serving

BIG = 1 << 60


def test_append_argument_errors_are_codes():
    L = _lib.load()

    def append(rows=16, ld=320, gain=16, rates=16, table=16, table_ld=4, width=4, lens=16, starts=16, n_seq=2, n=3, rank=256, rope=64, pages=9,
               page=64, dt=1, pool=16):
        return L.ethos_latent_append(rows, ld, gain, rates, table, table_ld, width, lens, starts, n_seq, n, rank, rope, pages, page, 1e-6, dt,
                                     pool, None)

    assert append(dt=2) == -1 and b"dtype" in L.ethos_last_error()
    for bad in (dict(n=-1), dict(n=1 << 31), dict(n_seq=-1), dict(n_seq=(1 << 20) + 1), dict(width=-1), dict(table_ld=3), dict(pages=0),
                dict(pages=1 << 31), dict(page=0), dict(rank=0), dict(rope=-8), dict(ld=312), dict(ld=324)):
        assert append(**bad) == -2, bad
    for bad in (dict(page=48), dict(page=1 << 17), dict(rank=260), dict(rope=60), dict(rank=520), dict(rope=136)):
        assert append(**bad) == -6, bad
    for name in ("rows", "gain", "rates", "table", "lens", "starts", "pool"):
        assert append(**{name: None}) == -3, name
    for name in ("rows", "gain", "pool"):
        assert append(**{name: 8}) == -4, name
    assert append(n=0, rows=None) == 0 and append(n_seq=0, lens=None) == 0 and L.ethos_last_error() == b""


def test_paged_attention_argument_errors_are_codes():
    L = _lib.load()

    def attend(q=16, w=16, pool=16, table=16, table_ld=4, width=4, lens=16, starts=16, rates=16, n=3, n_seq=2, H=16, rank=256, rope=64, nope=64,
               v=64, pages=9, page=64, dt=1, scale=0.1, ws=16, ws_bytes=BIG, out=16):
        return L.ethos_paged_attention(q, w, pool, table, table_ld, width, lens, starts, rates, n, n_seq, H, rank, rope, nope, v, pages, page, dt,
                                       scale, ws, ws_bytes, out, None)

    assert attend(dt=3) == -1
    for bad in (dict(n=-1), dict(n_seq=-1), dict(H=0), dict(H=1025), dict(nope=-1), dict(v=0), dict(nope=5000), dict(v=5000), dict(scale=0.0),
                dict(scale=-0.1), dict(scale=float("nan")), dict(scale=float("inf")), dict(n=(1 << 29) - 1), dict(table_ld=1)):
        assert attend(**bad) == -2, bad
    for bad in (dict(page=3), dict(rank=4), dict(rope=12), dict(rank=1024)):
        assert attend(**bad) == -6, bad
    for name in ("q", "w", "pool", "table", "lens", "starts", "rates", "ws", "out"):
        assert attend(**{name: None}) == -3, name
    for name in ("q", "w", "pool", "ws", "out"):
        assert attend(**{name: 8}) == -4, name
    need = L.ethos_paged_attention_workspace_bytes(3, 2, 16, 256, 64, 64, 64, 4, 64, 1)
    assert need > 0 and attend(ws_bytes=need - 1) == -5
    assert attend(n=0, q=None) == 0 and attend(n_seq=0, ws=None) == 0
    assert L.ethos_paged_attention_workspace_bytes(3, 2, 16, 256, 64, 64, 64, 4, 64, 9) == 256
    assert L.ethos_paged_attention_workspace_bytes(-3, 2, 16, 256, 64, 64, 64, 4, 64, 1) == 256


def test_paged_attention_refuses_more_rows_than_its_launches_take():
    L = _lib.load()
    for n, H, code in (((1 << 27) - 2047, 1, -2), ((1 << 23), 16, -2), ((1 << 27) - 2048, 1, -5), ((1 << 23) - 128, 16, -5), ((1 << 17) - 2, 1024, -5)):
        assert L.ethos_paged_attention(16, 16, 16, 16, 4, 4, 16, 16, 16, n, 2, H, 256, 64, 64, 64, 9, 64, 1, 0.1, 16, 0, 16, None) == code, (n, H)


def test_paged_attention_refuses_scales_beyond_its_arithmetic():
    L = _lib.load()
    for scale, code in ((3e38, -2), (1e36, -2), (1.01e35, -2), (1e35, -5), (1e-38, -5)):  # (-5: past the scale, to the workspace)
        assert L.ethos_paged_attention(16, 16, 16, 16, 4, 4, 16, 16, 16, 3, 2, 16, 256, 64, 64, 64, 9, 64, 1, scale, 16, 0, 16, None) == code, scale
    assert b"1e35" not in L.ethos_last_error()


def test_copy_pages_argument_errors_are_codes():
    L = _lib.load()
    arr = lambda *v: (ctypes.c_int32 * len(v))(*v)  # noqa: E731

    def copy(pool=16, blocks=2, block=4096, pages=4, page=1024, src=(0,), dst=(1,), n=1):
        return L.ethos_copy_pages(pool, blocks, block, pages, page, arr(*src), arr(*dst), n, None)

    for bad in (dict(blocks=-1), dict(blocks=65536), dict(pages=-1), dict(page=0), dict(page=3), dict(block=4095), dict(block=1024), dict(n=-1),
                dict(src=(4,)), dict(src=(-1,)), dict(dst=(4,)), dict(dst=(-1,))):
        assert copy(**bad) == -2, bad
    assert copy(pool=None) == -3 and copy(pool=17) == -4 and copy(n=0) == 0 and copy(blocks=0) == 0
    assert L.ethos_copy_pages(16, 2, 4096, 4, 1024, None, None, 1, None) == -3


def test_copy_pages_tells_the_same_page_by_its_number(monkeypatch):
    """Whatever kind of number it comes as."""
    numpy = pytest.importorskip("numpy")
    pairs = []
    monkeypatch.setattr(serving, "_check", lambda *a: None)
    monkeypatch.setattr(serving.hip, "copy_pages", lambda pool, src, dst: pairs.append((list(src), list(dst))))
    pool = torch.zeros(1, 9, 2)
    t = torch.tensor
    for src, dst in (([0, 1], [t(5), t(5)]), ([t(3)], [t(3)]), ([0, 1], [numpy.int64(5), t(5)]), ([3], [t(3)]), (t([1, 2]), [t(4), t(1)])):
        with pytest.raises(ValueError, match="twice"):
            ethos_amd.copy_pages(pool, src, dst)
    ethos_amd.copy_pages(pool, [t(0), numpy.int32(1)], (p for p in (t(5), 6)))
    ethos_amd.copy_pages(pool, numpy.array([2]), t([3], dtype=torch.int32))
    assert pairs == [([0, 1], [5, 6]), ([2], [3])]


def test_copy_pages_of_an_empty_pool_checks_the_pages():
    for shape in ((0, 5, 4, 8), (2, 5, 0, 8), (2, 5, 4, 0)):
        hip.copy_pages(torch.zeros(shape), [0, 3], [1, 4])
        hip.copy_pages(torch.zeros(shape), [], [])
        for src, dst in (([5], [1]), ([1], [5]), ([-1], [2]), ([2], [-1])):
            with pytest.raises(IndexError):
                hip.copy_pages(torch.zeros(shape), src, dst)
    with pytest.raises(IndexError):
        hip.copy_pages(torch.zeros(2, 0, 4, 8), [0], [1])


def test_copy_pages_names_too_many_blocks():
    """Not as pages outside the pool."""
    with pytest.raises(RuntimeError, match="65,535 blocks"):
        hip.copy_pages(torch.zeros(65536, 2, 1), [0], [1])


def test_verify_argument_errors_are_codes():
    L = _lib.load()

    def verify(logits=16, drafts=16, probs=16, pdt=0, counts=16, ua=16, us=16, b=3, m=2, V=50, t=1.0, dt=1, ws=16, ws_bytes=BIG, acc=16, tok=16):
        return L.ethos_verify(logits, drafts, probs, pdt, counts, ua, us, b, m, V, t, dt, ws, ws_bytes, acc, tok, None)

    assert verify(dt=2) == -1 and verify(pdt=5) == -1
    for bad in (dict(b=-1), dict(m=-1), dict(V=0), dict(t=-1.0), dict(t=1e-7), dict(t=1e7), dict(t=float("nan")), dict(b=1 << 30)):
        assert verify(**bad) == -2, bad
    for bad in (dict(m=256), dict(V=(1 << 24) + 1)):
        assert verify(**bad) == -6, bad
    for name in ("logits", "drafts", "ua", "us", "ws", "acc", "tok"):
        assert verify(**{name: None}) == -3, name
    assert verify(ws=8) == -4 and verify(logits=17) == -4 and verify(probs=18) == -4
    need = L.ethos_verify_workspace_bytes(3, 2, 50)
    assert need > 0 and verify(ws_bytes=need - 1) == -5
    assert verify(b=0, logits=None) == 0 and L.ethos_verify_workspace_bytes(3, 999, 50) == 256


def test_operators_have_no_cpu_path():
    t = torch.zeros(4, 4)
    i = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: ethos_amd.latent_append(t, t[0], t[None], i[None], i[:1], i[:2], t[0]),
                 lambda: ethos_amd.paged_attention(t[None], t, t[None], i[None], i[:1], i[:2], t[0], 1.0),
                 lambda: ethos_amd.copy_pages(t[None], [0], [1]),
                 lambda: ethos_amd.verify_drafts(t[None], i[None].long(), t, t[0])):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
    with pytest.raises(TypeError):
        ethos_amd.copy_pages([1], [0], [1])


# ------------------------------------------------------------------------------- the cache's books
def _book(monkeypatch, pages=12, page=4):
    """A cache on the host, with the page copies done there."""
    def copy(pool, src, dst):
        assert len(set(dst)) == len(dst) and not set(dst) & set(src)
        pool[:, dst] = pool[:, src]

    monkeypatch.setattr(serving, "copy_pages", copy)
    return serving.LatentCache(2, 8, 8, pages, page, torch.float32, "cpu")


def _write(c, batch, values):
    """Writes values[i] (a number a new token) of sequence i of the batch into the pool."""
    for i, vs in enumerate(values):
        first = int(batch.lens[i]) - len(vs)
        assert int(batch.starts[i + 1] - batch.starts[i]) == len(vs)
        for j, v in enumerate(vs):
            p = first + j
            c.pool[:, int(batch.table[i, p // c.page]), p % c.page] = v


def _read(c, seq):
    t = c.pages(seq)
    return [float(c.pool[0, t[p // c.page], p % c.page, 0]) for p in range(c.length(seq))]


def _consistent(c):
    users = [0] * len(c._users)
    for s in c._sequences.values():
        assert len(s.pages) == -(-s.length // c.page)
        for p in s.pages:
            users[p] += 1
    assert users == c._users
    assert sorted(c._free) == [p for p, n in enumerate(users) if n == 0]


def test_cache_is_made_on_the_device_it_is_given(monkeypatch):
    """A device's number too, zero among them."""
    asked = []

    def zeros(shape, dtype, device):
        asked.append(device)
        return torch.empty(shape, dtype=dtype)

    monkeypatch.setattr(serving.torch, "zeros", zeros)
    for device in (None, 0, 1, "cpu", torch.device("cuda", 0)):
        serving.LatentCache(1, 8, 8, 2, 4, torch.float32, device)
    assert asked == ["cuda", 0, 1, "cpu", torch.device("cuda", 0)]


def test_cache_keeps_every_sequence_its_tokens(monkeypatch):
    c = _book(monkeypatch)
    a, b = c.new(), c.new()
    _write(c, c.extend([a, b], [6, 3]), [[1, 2, 3, 4, 5, 6], [11, 12, 13]])
    assert c.length(a) == 6 and c.pages_free == 9
    f = c.fork(a)
    g = c.fork(a)
    assert c.pages(f) == c.pages(a) and c.pages_free == 9
    # all three write in the page that they share: two of them get a copy of it
    _write(c, c.extend([a, f, g], [1, 2, 3]), [[7], [70, 80], [700, 800, 900]])
    assert _read(c, a) == [1, 2, 3, 4, 5, 6, 7] and _read(c, f) == [1, 2, 3, 4, 5, 6, 70, 80]
    assert _read(c, g) == [1, 2, 3, 4, 5, 6, 700, 800, 900] and _read(c, b) == [11, 12, 13]
    _consistent(c)
    c.truncate(g, 4)
    c.truncate(f, 3)  # into a page that a and g have too
    _write(c, c.extend([f, b], [1, 0]), [[33], []])
    assert _read(c, f) == [1, 2, 3, 33] and _read(c, g) == [1, 2, 3, 4] and _read(c, a) == [1, 2, 3, 4, 5, 6, 7]
    _consistent(c)
    c.free(a)
    c.free(b)
    _consistent(c)
    used = c.compact()
    assert used == 2 and sorted(c.pages(f) + c.pages(g)) == [0, 1] and _read(c, f) == [1, 2, 3, 33] and _read(c, g) == [1, 2, 3, 4]
    _consistent(c)
    assert c.pages_free == 10 and c.compact() == 2
    with pytest.raises(KeyError):
        c.length(a)


def test_cache_compacts_shared_pages(monkeypatch):
    c = _book(monkeypatch, pages=9, page=2)
    a, b = c.new(), c.new()
    for k in range(4):
        _write(c, c.extend([a], [2]), [[k, k + 0.5]])
        _write(c, c.extend([b], [2]), [[10 + k, 10 + k + 0.5]])
    f = c.fork(b)
    c.free(a)
    assert c.compact() == 4
    assert sorted(c.pages(b)) == [0, 1, 2, 3] and c.pages(f) == c.pages(b)
    assert _read(c, b) == _read(c, f) == [10, 10.5, 11, 11.5, 12, 12.5, 13, 13.5]
    _consistent(c)


def test_cache_refuses_and_changes_nothing(monkeypatch):
    c = _book(monkeypatch, pages=3, page=4)
    a, b = c.new(), c.new()
    c.extend([a], [6])
    f = c.fork(a)
    before = (c.pages(a), c.pages(f), c.pages_free, c.length(a))
    for seqs, counts, error in (([a, b], [3, 1], RuntimeError), ([a, f], [3, 1], RuntimeError), ([b], [5], RuntimeError), ([a], [-1], ValueError),
                                ([a, a], [1, 1], ValueError), ([a], [1, 2], ValueError), ([99], [1], KeyError), ([a], [1.5], TypeError)):
        with pytest.raises(error):
            c.extend(seqs, counts)
        assert (c.pages(a), c.pages(f), c.pages_free, c.length(a)) == before, (seqs, counts)
    for length in (-1, 7):
        with pytest.raises(ValueError):
            c.truncate(a, length)
    for bad in (dict(blocks=0), dict(pages=0), dict(page=3), dict(page=0), dict(page=1 << 17), dict(rank=0), dict(rope=-2)):
        with pytest.raises(ValueError):
            serving.LatentCache(**{**dict(blocks=1, rank=8, rope=8, pages=2, page=4, device="cpu"), **bad})
    with pytest.raises(TypeError):
        serving.LatentCache(1, 8, 8, 2, 4, torch.float16, "cpu")
    e = c.extend([], [])
    assert e.table.shape[0] == 0 and e.starts.tolist() == [0]
    c.extend([b], [0])
    assert c.length(b) == 0


def test_cache_is_as_it_was_after_a_failure(monkeypatch):
    c = _book(monkeypatch, pages=8, page=4)
    a = c.new()
    _write(c, c.extend([a], [6]), [[1, 2, 3, 4, 5, 6]])
    f = c.fork(a)

    def refuse(*args):
        raise RuntimeError("refused")

    def state():
        return c.pages(a), c.pages(f), c.length(a), c.length(f), c.pages_free, sorted(c._free)

    before = state()
    with monkeypatch.context() as m:
        m.setattr(serving, "copy_pages", refuse)
        with pytest.raises(RuntimeError, match="refused"):
            c.extend([f, a], [1, 9])
    assert state() == before
    _consistent(c)
    with monkeypatch.context() as m:
        m.setattr(c, "_batch", refuse)
        with pytest.raises(RuntimeError, match="refused"):
            c.extend([a], [9])
    assert (c.length(a), c.length(f)) == (6, 6) and _read(c, a) == _read(c, f) == [1, 2, 3, 4, 5, 6]
    _consistent(c)
    with pytest.raises(TypeError):
        c.truncate(a, 2.0)


def test_cache_against_a_plain_one(monkeypatch):
    """Random steps, with lists of numbers beside the cache."""
    import random

    rng = random.Random(5)
    c = _book(monkeypatch, pages=40, page=4)
    plain = {}
    for step in range(400):
        do = rng.choice(["new", "extend", "extend", "extend", "fork", "truncate", "free", "compact"])
        live = list(plain)
        if do == "new" or not live:
            plain[c.new()] = []
        elif do == "extend":
            seqs = rng.sample(live, min(len(live), rng.randint(1, 4)))
            values = [[rng.randint(1, 999) for _ in range(rng.randint(0, 9))] for _ in seqs]
            try:
                batch = c.extend(seqs, [len(v) for v in values])
            except RuntimeError:
                c.free(live[0])
                del plain[live[0]]
                continue
            _write(c, batch, values)
            for q, v in zip(seqs, values):
                plain[q] += v
        elif do == "fork":
            q = rng.choice(live)
            plain[c.fork(q)] = list(plain[q])
        elif do == "truncate":
            q = rng.choice(live)
            n = rng.randint(0, len(plain[q]))
            c.truncate(q, n)
            del plain[q][n:]
        elif do == "free":
            q = rng.choice(live)
            c.free(q)
            del plain[q]
        else:
            used = c.compact()
            assert all(p < used for q in plain for p in c.pages(q))
        _consistent(c)
        for q, v in plain.items():
            assert _read(c, q) == v
