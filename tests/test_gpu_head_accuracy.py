"""The token head's results entry by entry against their definitions in 64 bits: small gradients beside large ones, masks of
the lowest value and of infinity in the table, values of very different sizes in one tensor.

Bounds are counted from the roundings, for each logit and each entry by itself: u = eps / 2 of a type is the most that
one rounding to it is off, relative to the value."""
import pytest
import torch  # before libpst loads: one HIP runtime serves both

from pst_amd import head

pytestmark = pytest.mark.gpu

DEV = "cuda"
U32 = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# half the smallest step of the type
LEAST = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
TYPES = [torch.bfloat16, torch.float16, torch.float32]
SIXTEEN = [torch.bfloat16, torch.float16]


def make(rows, vocab, width, dtype, seed=0, ignored=0.2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, width, generator=g, device=DEV).to(dtype)
    w = (torch.randn(vocab, width, generator=g, device=DEV) * width ** -0.5).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    t[torch.rand(rows, generator=g, device=DEV) < ignored] = -100
    gl = torch.rand(rows, generator=g, device=DEV) + 0.5
    return x, w, t, gl


def with_bias(x, w):
    """A column of ones beside a column of biases: what sets single ids' logits."""
    x, w = x.clone(), w.clone()
    x[:, -1], w[:, -1] = 1, 0
    return x, w


def product(a, b, terms, u=U32):
    """What a product of 64-bit matrices is, and what `terms` additions in 32 bits may put it off."""
    mag = a.abs() @ b.abs()
    return a @ b, torch.where(mag.isfinite(), mag, 0.0) * u * (terms + 2)


def check_loss(x, w, t):
    loss, lse = head.token_loss(x, w, t)
    l, off = product(x.double(), w.double().T, x.shape[1])
    want_lse = torch.logsumexp(l, 1)
    p = torch.exp(l - want_lse[:, None])
    keep = t != -100
    at = torch.where(keep, t, 0)[:, None]
    want = torch.where(keep, want_lse - l.gather(1, at)[:, 0], 0.0)
    # the logits' errors as they count; chains of at most 128 + V / 1024 + 40 additions of exponentials of 4 roundings each
    # (those of the argument count (l - max) times, which its exponential outruns); the results' own roundings
    tol = (p * off).sum(1) + (180 + w.shape[0] / 1024) * U32 + 8 * U32 * (want_lse.abs() + 1)
    assert ((lse.double() - want_lse).abs() <= tol).all()
    assert ((loss.double() - want).abs() <= tol + off.gather(1, at)[:, 0] + 4 * U32 * want.abs())[keep].all()
    assert (loss[~keep] == 0).all()
    return loss, lse


def check_grad(x, w, t, gl, lse=None, columns=slice(None)):
    """Both gradients, each entry (of `columns`) within what its own terms' roundings may put it off."""
    if lse is None:
        lse = head.token_loss(x, w, t)[1]
    dx, dw = head.token_loss_grad(x, w, t, lse, gl)
    dt, n, v, d = x.dtype, x.shape[0], w.shape[0], x.shape[1]
    l, off = product(x.double(), w.double().T, d)
    keep = t != -100
    z = l - lse.double()[:, None]
    p = torch.where(keep[:, None], torch.exp(z), 0.0)
    slope = p.clone()
    slope[torch.arange(n, device=DEV)[keep], t[keep]] -= 1
    c = torch.where(keep, gl.double(), 0.0)[:, None]
    slope *= c
    # the exponential of l - lse: the logit's error, and 4 roundings of the difference (p z is nothing where p is 0)
    z = torch.where(p > 0, z, 0.0)
    err = c.abs() * p * (torch.expm1(off.clamp(max=700)).where(p > 0, 0.0) + 4 * U32 * (z.abs() + 2)) + slope.abs() * 4 * U32
    # 16-bit types: the slope as a sum of two bf16 halves (2^-16); f16: without the product of two low halves (2^-16)
    halves = 0.0 if dt == torch.float32 else 2.0 ** -16
    # (the hardware's exponential of less than the smallest normal number, 2^-126, is 0: never more than that off)
    err = err + slope.abs() * halves + c.abs() * 2.0 ** -126
    left = 2.0 ** -16 if dt == torch.float16 else 0.0
    passes = {torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}[dt]
    for got, s, e, other, terms in ((dx, slope, err, w, v), (dw, slope.T, err.T, x, n)):
        o = torch.where(keep[:, None], x, 0).double() if other is x else w.double()
        want = s @ o
        a = torch.where(o.isfinite(), o.abs(), 0.0)
        tol = e @ a + (s.abs() @ a) * (U32 * (passes * terms + 16) + left) + want.abs() * U[dt] * 1.01 + LEAST[dt]
        # what is past the type's largest value is an infinity: an entry that its bound leaves there may be one, of its sign
        over = (want.abs() + tol > torch.finfo(dt).max) & (got.double() == want.sign() * torch.inf)
        bad = (((got.double() - want).abs() > tol) & ~over)[:, columns]
        assert not bad.any(), (bad.sum().item(), ((got.double() - want).abs() / tol)[:, columns].max().item())
        assert not got[:, columns].isnan().any()
    assert (dx[~keep] == 0).all()
    return dx, dw


# the slope g (p - 1) is not rounded to the operands' 16 bits: sums of many slopes keep what cancels between them
@pytest.mark.parametrize("dtype", SIXTEEN, ids=str)
@pytest.mark.parametrize("rows,vocab,width", [(40, 300, 64), (600, 700, 136), (2049, 4099, 72), (1100, 2100, 1000), (900, 130, 8)])
def test_slopes_keep_their_bits(rows, vocab, width, dtype):
    check_grad(*make(rows, vocab, width, dtype, seed=1))


# weights of positions over six decades: each position's gradient is as good as if it were alone
@pytest.mark.parametrize("dtype", SIXTEEN, ids=str)
@pytest.mark.parametrize("rows,vocab,width", [(200, 64003, 64), (1100, 4099, 96)])
def test_weights_of_very_different_sizes(rows, vocab, width, dtype):
    x, w, t, _ = make(rows, vocab, width, dtype, seed=2)
    w = (w.float() + 0.1).to(dtype)  # (rows that do not cancel: the softmax's part of the gradient counts)
    gl = 10.0 ** torch.linspace(-4, 2, rows, device=DEV)
    check_grad(x, w, t, gl)
    check_grad(x, w, t, gl.flip(0))


# an id that all positions find improbable: its row's gradient has as many right digits as any
@pytest.mark.parametrize("dtype,bias,weight", [(torch.bfloat16, -40, 1.0), (torch.bfloat16, -60, 1.0), (torch.float16, -24, 6e4)], ids=str)
@pytest.mark.parametrize("rows,vocab,width", [(60, 500, 64), (1200, 2100, 80)])
def test_improbable_ids(rows, vocab, width, dtype, bias, weight):
    x, w, t, gl = make(rows, vocab, width, dtype, seed=3)
    x, w = with_bias(x, w)
    w[5, -1] = bias
    t[t == 5] = 6
    _, dw = check_grad(x, w, t, gl * weight / 1.5)
    # float16: e^-24 / 500 ids, times 4e4 and a sum of 48 of either sign, is 2e-8, less than the smallest step of 6e-8
    assert dtype == torch.float16 or (dw[5] != 0).all()


# in 32 bits too: each value keeps its digits whatever else its row, its tensor or the weights of positions hold
@pytest.mark.parametrize("rows,vocab,width", [(40, 300, 64), (600, 700, 136), (2049, 4099, 72), (1100, 2100, 333), (900, 130, 8)])
def test_32_bits(rows, vocab, width):
    x, w, t, gl = make(rows, vocab, width, torch.float32, seed=1)
    check_loss(x, w, t)
    check_grad(x, w, t, gl)


@pytest.mark.parametrize("rows,vocab,width", [(200, 64003, 64), (1100, 4099, 96)])
def test_32_bit_weights_and_rows_of_very_different_sizes(rows, vocab, width):
    x, w, t, _ = make(rows, vocab, width, torch.float32, seed=2)
    w += 0.1
    gl = 10.0 ** torch.linspace(-9, 6, rows, device=DEV)
    check_grad(x, w, t, gl)
    check_grad(x, w, t, gl.flip(0))
    sizes = 10.0 ** torch.linspace(-6, 1, rows, device=DEV)[:, None]
    check_grad(x * sizes, w, t, gl)
    # one column of hidden a million million times the others', with nothing in the table beside it
    x[:, 0], w[:, 0] = 1e12, 0
    check_loss(x, w, t)
    check_grad(x, w, t, gl, columns=slice(1, None))


@pytest.mark.parametrize("bias", [-40, -80])
@pytest.mark.parametrize("rows,vocab,width", [(60, 500, 64), (1200, 2100, 80)])
def test_32_bit_improbable_ids(rows, vocab, width, bias):
    x, w, t, gl = make(rows, vocab, width, torch.float32, seed=3)
    x, w = with_bias(x, w)
    w[5, -1] = bias
    t[t == 5] = 6
    _, dw = check_grad(x, w, t, gl)
    assert (dw[5] != 0).all()


MASKED = [(40, 300, 96), (600, 700, 128), (2049, 4099, 160), (1200, 2100, 333), (3, 70, 64)]


# ids that are not allowed: their bias is a large negative number, as large as the type has
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("mask", ["least", -1e30, -1e9, -1e4])
@pytest.mark.parametrize("rows,vocab,width", MASKED)
def test_masks_of_large_numbers(rows, vocab, width, mask, dtype):
    least = torch.finfo(dtype).min
    x, w, t, gl = make(rows, vocab, width, dtype, seed=4)
    x, w = with_bias(x, w)
    w[[5, vocab - 1], -1] = least if mask == "least" else max(mask, least)
    t[(t == 5) | (t == vocab - 1)] = 6
    x[::3, -1] = 0  # (positions that allow them)
    _, lse = check_loss(x, w, t)
    check_grad(x, w, t, gl, lse)


# the same with -inf: probability 0, and nothing else of the position's
# (widths of 72 and 100: rows read in place that end inside a K-step, with the infinity in their last 16 bytes)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,width", MASKED + [(600, 700, 72), (600, 700, 100), (2100, 4160, 8), (70, 20000, 20)])
def test_masks_of_infinity(rows, vocab, width, dtype):
    x, w, t, gl = make(rows, vocab, width, dtype, seed=5)
    x, w = with_bias(x, w)
    w[[5, vocab - 1], -1] = -torch.inf
    t[(t == 5) | (t == vocab - 1)] = 6
    _, lse = check_loss(x, w, t)
    assert lse.isfinite().all()
    # (the bias column of hidden's gradient is a sum over 0 (-inf))
    dx, _ = check_grad(x, w, t, gl, lse, columns=slice(0, -1))
    assert not dx[t != -100, -1].isfinite().any()


# more positions than a piece of the logits' gradient holds: the table's gradient is summed over the pieces
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,width", [(20000, 9001, 40), (8193, 16000, 24), (299000, 50, 16)])
def test_pieces_of_the_positions(rows, vocab, width, dtype):
    x, w, t, gl = make(rows, vocab, width, dtype, seed=6)
    lse = head.token_loss(x, w, t)[1]
    dx, dw = check_grad(x, w, t, gl, lse)
    a, none = head.token_loss_grad(x, w, t, lse, gl, need_weight=False)
    assert none is None and torch.equal(a, dx)
    none, b = head.token_loss_grad(x, w, t, lse, gl, need_hidden=False)
    assert none is None and torch.equal(b, dw)


# a position whose mask leaves no id: nothing to divide by, and it says so; the others do not notice
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,width", [(3, 70, 64), (300, 700, 72), (1200, 2100, 100)])
def test_a_mask_that_leaves_nothing(rows, vocab, width, dtype):
    x, w, t, _ = make(rows, vocab, width, dtype, seed=7)
    x, w = with_bias(x, w)
    x[:, -1] = 0
    whole_loss, whole_lse = head.token_loss(x, w, t)
    w[:, -1] = -torch.inf
    x[:, -1] = 1
    loss, lse = head.token_loss(x, w, t)
    assert (lse == -torch.inf).all() and loss[t != -100].isnan().all() and (loss[t == -100] == 0).all()
    w[:, -1] = torch.where(torch.arange(vocab, device=DEV) % 2 == 0, -torch.inf, 0.0).to(dtype)
    loss, lse = head.token_loss(x, w, t)
    l = x[:, :-1].double() @ w[1::2, :-1].double().T
    off = (x[:, :-1].double().abs() @ w[1::2, :-1].double().abs().T).amax(1) * U32 * (width + 2)
    assert ((lse.double() - torch.logsumexp(l, 1)).abs() <= off + (200 + vocab / 1024) * U32 + 8 * U32 * (lse.abs() + 1)).all()
    assert (loss[(t != -100) & (t % 2 == 0)] == torch.inf).all() and whole_loss.isfinite().all() and whole_lse.isfinite().all()
