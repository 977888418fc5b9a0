"""The serving operators' refusals that need no GPU: argument errors of the C-ABI come back as codes
before anything is enqueued, and the Python entry points name what is wrong."""
import ctypes

import pytest
import torch

import ethos_amd
from ethos_amd import _lib

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
