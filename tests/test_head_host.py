"""The token head's checks of arguments, without a GPU: the C entry points refuse before they touch a device, the Python
layer before it calls them; and the shape rules of its workspaces."""
import ctypes

import pytest
import torch  # before libpst loads: one HIP runtime serves both

from pst_amd import _native, head

F32, BF16, F16 = 0, 1, 2
BUF = ctypes.create_string_buffer(4096)
P = (ctypes.addressof(BUF) + 255) // 256 * 256  # 256-byte aligned


def loss(device=0, type=BF16, x=P, ldx=64, w=P, ldw=64, rows=4, vocab=8, width=64, t=P, bits=64, ignore=-100, out=P, lse=P, ws=P, n=1 << 40):
    return _native.lib().pst_token_loss(device, type, x, ldx, w, ldw, rows, vocab, width, t, bits, ignore, out, lse, ws, n, None)


def grad(type=BF16, x=P, ldx=64, w=P, ldw=64, rows=4, vocab=8, width=64, t=P, bits=64, lse=P, g=P, dx=P, lddx=64, dw=P, lddw=64, ws=P, n=1 << 40):
    return _native.lib().pst_token_loss_grad(0, type, x, ldx, w, ldw, rows, vocab, width, t, bits, -100, lse, g, dx, lddx, dw, lddw, ws, n, None)


def scores(type=BF16, x=P, ldx=64, w=P, ldw=64, s=P, rows=4, vocab=8, width=64, ot=F32, out=P, ldo=8, ws=P, n=1 << 40):
    return _native.lib().pst_token_scores_i8(0, type, x, ldx, w, ldw, s, rows, vocab, width, ot, out, ldo, ws, n, None)


def quant(type=BF16, x=P, ldx=64, rows=4, width=64, q=P, ldq=64, s=P):
    return _native.lib().pst_quantize_rows(0, type, x, ldx, rows, width, q, ldq, s, None)


BAD = [dict(type=3), dict(type=-1), dict(rows=-1), dict(vocab=0), dict(width=0), dict(ldx=63), dict(ldw=63), dict(x=None), dict(w=None)]


@pytest.mark.parametrize("bad", BAD + [dict(x=P + 1), dict(w=P + 1), dict(t=None), dict(bits=16), dict(t=P + 4), dict(out=None), dict(lse=None),
                                       dict(lse=P + 2), dict(ws=None), dict(ws=P + 16), dict(n=16), dict(type=F32, x=P + 2)])
def test_loss_refuses(bad):
    assert loss(**bad) == _native.PST_E_INVALID
    assert _native.lib().pst_head_error()


@pytest.mark.parametrize("bad", BAD + [dict(t=None), dict(bits=8), dict(lse=None), dict(g=None), dict(lddx=63), dict(lddw=1), dict(dx=P + 1), dict(dw=P + 1),
                                       dict(ws=P + 128), dict(n=0)])
def test_grad_refuses(bad):
    assert grad(**bad) == _native.PST_E_INVALID


@pytest.mark.parametrize("bad", BAD + [dict(s=None), dict(ot=3), dict(out=None), dict(out=P + 2), dict(ldo=7), dict(ws=None), dict(n=1)])
def test_scores_refuse(bad):
    assert scores(**bad) == _native.PST_E_INVALID


@pytest.mark.parametrize("bad", [dict(type=5), dict(rows=-1), dict(width=0), dict(ldx=3), dict(ldq=63), dict(x=None), dict(q=None), dict(s=None), dict(s=P + 1)])
def test_quantize_refuses(bad):
    assert quant(**bad) == _native.PST_E_INVALID


@pytest.mark.parametrize("fn,bad", [(loss, dict(rows=1 << 31)), (loss, dict(vocab=1 << 31)), (loss, dict(width=1 << 21, ldx=1 << 21, ldw=1 << 21)),
                                    (grad, dict(ldx=1 << 22)), (scores, dict(width=131073, ldx=131073, ldw=131073)), (quant, dict(rows=1 << 31))])
def test_too_large(fn, bad):
    assert fn(**bad) == _native.PST_E_TOO_LARGE


def test_nothing_to_do_is_no_error():
    assert loss(rows=0, x=None, t=None) == _native.PST_OK
    assert grad(dx=None, dw=None) == _native.PST_OK
    assert grad(rows=0, dw=None, x=None, t=None, lse=None, g=None) == _native.PST_OK
    assert scores(rows=0, x=None) == _native.PST_OK
    assert quant(rows=0, x=None) == _native.PST_OK


def test_without_a_device_the_runtime_s_error_is_named():
    if _native.device_count() > 0:
        pytest.skip("a HIP device is visible")
    for fn in (loss, grad, scores, quant):
        assert fn() == _native.PST_E_HIP
        assert b"device 0" in _native.lib().pst_head_error()


def test_workspaces():
    L = _native.lib()
    for fn in (L.pst_token_loss_workspace, L.pst_token_loss_grad_workspace):
        a = fn(BF16, P, 64, P, 64, 100, 1000, 64)
        assert a > 0
        assert fn(BF16, P, 65, P, 65, 100, 1000, 64) > a  # copies
        assert fn(F32, P, 64, P, 64, 100, 1000, 64) > a   # splits
        assert fn(BF16, P, 64, P, 64, 100, 0, 64) < 0
    # whatever the vocabulary: a piece of the logits' gradient, hidden's copy and up to eight partial sums of its gradient
    for vocab in (64000, 640000):
        n = L.pst_token_loss_grad_workspace(BF16, P, 1024, P, 1024, 8192, vocab, 1024)
        assert n <= (288 << 20) + 8192 * 1024 * (2 + 8 * 4) + 4096


def test_python_layer_refuses():
    x, w, t = torch.zeros(4, 8), torch.zeros(16, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        head.token_loss(x, w, t)
    with pytest.raises(ValueError, match="GPU"):
        head.token_loss_grad(x, w, t, torch.zeros(4), torch.zeros(4))
    with pytest.raises(ValueError, match="GPU"):
        head.quantize_rows(x)
    with pytest.raises(ValueError, match="GPU"):
        head.token_scores_int8(x, w.to(torch.int8), torch.zeros(16))


def test_strides_are_checked():
    m = torch.zeros(6, 8)
    assert head._matrix(m[:, :4], "m") == (m.data_ptr(), 8)
    assert head._matrix(m[:1], "m") == (m.data_ptr(), 8)
    with pytest.raises(ValueError, match="column stride"):
        head._matrix(m.t(), "m")
    with pytest.raises(ValueError, match="overlapping"):
        head._matrix(m[:1].expand(4, 8), "m")
    with pytest.raises(ValueError, match="dimensions"):
        head._matrix(m[0], "m")
    with pytest.raises(ValueError, match="vector"):
        head._vector(m[:, 0], "v", 6, m.device)


def test_another_thread_s_first_call_sees_all_of_the_set_up(monkeypatch):
    order = []

    class Watched(dict):
        def __setitem__(self, key, value):
            order.append(head._torch_module)
            super().__setitem__(key, value)

    monkeypatch.setattr(head, "_torch_module", None)
    monkeypatch.setattr(head, "_target_bits", Watched())
    assert head._torch() is torch
    # while the table of target types is filled nobody is told that it is there
    assert order and all(m is None for m in order) and set(head._target_bits) == {torch.int32, torch.int64}


def test_workspaces_of_sizes_that_are_too_large():
    L = _native.lib()
    for fn in ("pst_token_loss_workspace", "pst_token_loss_grad_workspace", "pst_token_scores_i8_workspace"):
        for rows, vocab, width in ((1 << 31, 8, 64), (4, 1 << 31, 64), (4, 8, 1 << 21)):
            args = (BF16, P, max(width, 64), P, max(width, 64), rows, vocab, width)
            assert getattr(L, fn)(*args) == _native.PST_E_TOO_LARGE
            assert b"over 2^30" in L.pst_head_error()
            with pytest.raises(NotImplementedError, match="2\\^30"):
                head._workspace_bytes(fn, *args)


@pytest.mark.parametrize("type,size", [(BF16, 2), (F16, 2), (F32, 4)])
def test_the_gradient_s_workspace_does_not_grow_with_the_positions(type, size):
    L = _native.lib()
    for vocab, width in ((64003, 1024), (4099, 1024), (432, 256)):
        # pieces of the logits' gradient, and of the positions that have one: copies of hidden (float16: and halves) and
        # up to eight sums of its gradient; up to two sums of all of the weight's (float16: and its halves)
        span = max(8192, (288 << 20) // (4 * ((vocab + 255) // 256 * 256)))
        most = (288 << 20) + span * width * (size + 4 + 4 * 8) + vocab * width * 4 * 3 + 4096
        for rows in (131072, 524288, 1 << 24):
            assert 0 < L.pst_token_loss_grad_workspace(type, P, width, P, width, rows, vocab, width) <= most
