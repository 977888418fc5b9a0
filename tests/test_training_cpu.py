"""The training operators' refusals that need no GPU: argument errors of the C-ABI come back as codes
before anything is enqueued, and the Python entry points name what is wrong."""
import ctypes

import pytest
import torch

import ethos_amd
from ethos_amd import _lib


def test_linear_ce_argument_errors_are_codes():
    L = _lib.load()
    big = 1 << 40

    def ce(h=16, ldh=64, w=16, labels=16, n=4, d=64, V=9, ignore=-100, red=0, dt=1, st=16, st_bytes=big, ex=None, ex_bytes=0,
           ws=16, ws_bytes=big, loss=16):
        return L.ethos_linear_ce(h, ldh, w, labels, n, d, V, ignore, red, dt, st, st_bytes, ex, ex_bytes, ws, ws_bytes, loss, None)

    assert ce(dt=2) == -1 and b"dtype" in L.ethos_last_error()
    for bad in (dict(n=-1), dict(n=(1 << 30) + 1), dict(d=0), dict(V=0), dict(V=(1 << 30) + 1), dict(red=3), dict(red=-1), dict(ldh=56)):
        assert ce(**bad) == -2, bad
    for bad in (dict(d=60), dict(d=32776, ldh=32776), dict(ldh=68), dict(ldh=66, dt=0)):
        assert ce(**bad) == -6, bad
    for name in ("h", "w", "labels", "st", "ws", "loss"):
        assert ce(**{name: None}) == -3, name
        if name not in ("labels", "loss"):
            assert ce(**{name: 24}) == -4, name
    assert ce(st_bytes=L.ethos_linear_ce_state_bytes(4, 64, 1) - 1) == -5
    assert ce(ws_bytes=L.ethos_linear_ce_workspace_bytes(4, 64, 9, 1) - 1) == -5
    assert ce(ex=16, ex_bytes=L.ethos_linear_ce_exps_bytes(4, 9, 1) - 1) == -5 and ce(ex=24, ex_bytes=big) == -4
    assert ce(ex=16, ex_bytes=big, dt=0) == -6 and L.ethos_linear_ce_exps_bytes(4, 9, 0) == 0
    assert ce(n=0, h=None) == 0 and L.ethos_last_error() == b""

    def grad(st=16, st_bytes=big, ex=None, ex_bytes=0, w=16, dl=16, n=4, d=64, V=9, red=0, dt=1, ws=16, ws_bytes=big, dh=16, dw=16):
        return L.ethos_linear_ce_grad(st, st_bytes, ex, ex_bytes, w, dl, n, d, V, red, dt, ws, ws_bytes, dh, dw, None)

    assert grad(dt=7) == -1 and grad(V=0) == -2 and grad(red=5) == -2 and grad(d=4) == -6
    for name in ("st", "w", "dl", "ws"):
        assert grad(**{name: None}) == -3, name
    for name in ("st", "w", "ws", "dh", "dw"):
        assert grad(**{name: 8}) == -4, name
    assert grad(ws_bytes=L.ethos_linear_ce_grad_workspace_bytes(4, 64, 9, 1, 0) - 1) == -5 and grad(st_bytes=8) == -5
    assert grad(ex=16, ex_bytes=8) == -5 and grad(ex=24, ex_bytes=big) == -4 and grad(ex=16, ex_bytes=big, dt=0) == -6
    assert grad(n=0, w=None) == 0 and grad(dh=None, dw=None) == 0


def test_linear_ce_refuses_more_rows_than_its_launches_have_threads_for():
    L = _lib.load()
    big, most = 1 << 60, (1 << 26) - 256
    for n, code in ((most, -3), (most + 1, -2), (1 << 26, -2), (1 << 30, -2)):
        assert L.ethos_linear_ce(None, 8, 16, 16, n, 8, 9, -100, 0, 1, 16, big, None, 0, 16, big, 16, None) == code, n
        assert L.ethos_linear_ce_grad(None, big, None, 0, 16, 16, n, 8, 9, 0, 1, 16, big, 16, 16, None) == code, n
    assert L.ethos_linear_ce_state_bytes(most, 8, 1) > most and L.ethos_linear_ce_state_bytes(most + 1, 8, 1) == 256


def test_capture_id_needs_a_place_for_it():
    L = _lib.load()
    assert L.ethos_capture_id(None, None) == -3 and b"null" in L.ethos_last_error()


def test_embedding_balance_and_clip_argument_errors_are_codes():
    L = _lib.load()
    big, top = 1 << 40, 2 ** 31 - 1
    emb = lambda ids=16, w=16, n=4, d=8, V=9, dt=1, out=16: L.ethos_embedding(ids, 1, w, n, d, V, 1.0, -1, dt, out, None, None)  # noqa: E731
    assert emb(dt=3) == -1 and emb(n=-1) == -2 and emb(d=0) == -2 and emb(V=0) == -2 and emb(V=top) == -2 and emb(n=top) == -2
    assert emb(ids=None) == -3 and emb(w=None) == -3 and emb(out=None) == -3 and emb(w=17) == -4 and emb(out=18, dt=0) == -4
    assert emb(n=0, ids=None) == 0

    def egrad(ids=16, dy=16, n=4, d=8, V=9, dt=1, ws=16, ws_bytes=big, dw=16):
        return L.ethos_embedding_grad(ids, dy, n, d, V, 1.0, dt, ws, ws_bytes, dw, None)

    assert egrad(dt=3) == -1 and egrad(V=0) == -2 and egrad(ids=None) == -3 and egrad(dy=None) == -3 and egrad(dw=None) == -3
    assert egrad(dy=24) == -4 and egrad(dw=24) == -4 and egrad(ws=8) == -4
    assert egrad(ws_bytes=L.ethos_embedding_grad_workspace_bytes(4, 8, 9) - 1) == -5

    def bal(g=16, ids=16, n=4, H=2, k=3, E=5, dt=1, ws=16, ws_bytes=big, c=16, loss=16):
        return L.ethos_balance(g, ids, 1, n, H, k, E, dt, ws, ws_bytes, c, loss, None)

    assert bal(dt=9) == -1 and bal(n=-1) == -2 and bal(H=0) == -2 and bal(k=0) == -2 and bal(E=0) == -2 and bal(E=top + 1) == -2
    assert bal(n=1 << 20, H=1 << 10, k=4) == -2 and bal(n=top, H=top, k=top) == -2
    for name in ("g", "ids", "ws", "c", "loss"):
        assert bal(**{name: None}) == -3, name
    assert bal(ws=8) == -4 and bal(g=17) == -4 and bal(ws_bytes=L.ethos_balance_workspace_bytes(4, 2, 3, 5) - 1) == -5
    bgrad = lambda ids=16, c=16, dl=16, n=4, dt=1, out=16: L.ethos_balance_grad(ids, 1, c, dl, n, 2, 3, 5, dt, out, None)  # noqa: E731
    assert bgrad(dt=9) == -1 and bgrad(n=-1) == -2 and bgrad(out=17) == -4 and bgrad(n=0, ids=None) == 0
    for name in ("ids", "c", "dl", "out"):
        assert bgrad(**{name: None}) == -3, name

    ptr, i64, i32 = ctypes.c_void_p * 2, ctypes.c_int64 * 2, ctypes.c_int32 * 2

    def clip(a=(16, 32), b=(16, 32), sizes=(3, 4), dts=(1, 0), n=2, ws=16, ws_bytes=big, total=16):
        return L.ethos_clip_grads(ptr(*a), ptr(*b), i64(*sizes), i32(*dts), n, 0, 1.0, ws, ws_bytes, total, None)

    assert clip(n=-1) == -2 and clip(sizes=(3, -4)) == -2 and clip(sizes=(3, (1 << 40) + 1)) == -2 and clip(dts=(1, 2)) == -1
    assert clip(a=(16, None)) == -3 and clip(b=(None, 16)) == -3 and clip(ws=None) == -3 and clip(total=None) == -3
    assert clip(a=(17, 32)) == -4 and clip(b=(16, 34)) == -4 and clip(ws=8) == -4 and clip(ws_bytes=16) == -5


def test_entry_points_refuse_host_tensors():
    h, l = torch.zeros(4, 16), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: ethos_amd.linear_cross_entropy(h, h, l), lambda: ethos_amd.embedding(l, h),
                 lambda: ethos_amd.balance_loss(h, l, 4), lambda: ethos_amd.clip_grads([h], 1.0)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
    with pytest.raises(TypeError):
        ethos_amd.linear_cross_entropy(None, h, l)


def _calls(f, i):
    """The four entry points with a float tensor f [4, 8] in each differentiable place, and whole numbers i [4, 8]."""
    ids = i.view(-1)[:4]
    return (lambda: ethos_amd.linear_cross_entropy(f, f.detach(), ids), lambda: ethos_amd.linear_cross_entropy(f.detach(), f, ids),
            lambda: ethos_amd.embedding(ids, f), lambda: ethos_amd.balance_loss(f, i, 4), lambda: ethos_amd.clip_grads([f], 1.0),
            lambda: ethos_amd.clip_grads([f.detach()], 1.0, out=[f]))


@pytest.mark.parametrize("grad", [False, True])
def test_entry_points_refuse_forward_mode_derivatives(grad):
    i = torch.zeros(4, 8, dtype=torch.int64)
    with torch.autograd.forward_ad.dual_level():
        f = torch.autograd.forward_ad.make_dual(torch.ones(4, 8, requires_grad=grad), torch.ones(4, 8))
        # (torch's detach keeps the tangent: both operands of the loss have one)
        for call in _calls(f, i):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        # without a tangent it goes on, here to the refusal of host tensors
        for call in _calls(torch.ones(4, 8), i):
            with pytest.raises(RuntimeError, match="HIP device"):
                call()


def test_entry_points_refuse_tracing():
    i = torch.zeros(4, 8, dtype=torch.int64)
    for k in range(len(_calls(torch.ones(4, 8), i))):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(lambda f: _calls(f, i)[k](), (torch.ones(4, 8),))
