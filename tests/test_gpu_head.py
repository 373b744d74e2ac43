"""The token head's operators on the GPU against their definitions in 64 bits, with bounds counted from the roundings:
u = eps / 2 of a type is the most that one rounding to it is off, relative to the value."""
import pytest
import torch  # before libpst loads: one HIP runtime serves both

from pst_amd import _native, head

pytestmark = pytest.mark.gpu

DEV = "cuda"
U32 = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(rows, vocab, width, dtype, seed=0, pad=0, wpad=0, ignored=0.2, tdtype=torch.int64):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, width + pad, generator=g, device=DEV).to(dtype)[:, :width]
    w = (torch.randn(vocab, width + wpad, generator=g, device=DEV) * width ** -0.5).to(dtype)[:, :width]
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    t[torch.rand(rows, generator=g, device=DEV) < ignored] = -100
    gl = torch.rand(rows, generator=g, device=DEV) + 0.5
    return x, w, t.to(tdtype), gl


def logit_bound(x, w):
    """What a logit may be off: sums of `width` (32-bit inputs: 3 width, of split values, 8 u) terms in 32 bits."""
    x, w = x.double(), w.double()
    d = x.shape[1]
    b = (x.abs() @ w.abs().T).amax(1) * U32 * (d + 2)
    return b * 3 + (x.abs() @ w.abs().T).amax(1) * 8 * U32


def defined_loss(x, w, t, ignore=-100):
    l = x.double() @ w.double().T
    lse = torch.logsumexp(l, 1)
    keep = t != ignore
    at = l.gather(1, torch.where(keep, t, 0).long()[:, None])[:, 0]
    return torch.where(keep, lse - at, 0.0), lse


def check_loss(x, w, t, **kw):
    loss, lse = head.token_loss(x, w, t, **kw)
    want, want_lse = defined_loss(x, w, t, **{"ignore": kw["ignore_index"]} if kw else {})
    # the sum of exponentials: chains of at most 128 + V / 1024 + 40 additions, and 4 roundings in each exponent
    rel = (170 + w.shape[0] / 1024) * U32
    tol = logit_bound(x, w) + rel + 8 * U32 * (want_lse.abs() + 1)
    assert ((lse.double() - want_lse).abs() <= tol).all()
    assert ((loss.double() - want).abs() <= 2 * tol).all()
    assert (loss[t == kw.get("ignore_index", -100)] == 0).all()
    return loss, lse


def defined_grad(x, w, t, lse, gl, ignore=-100):
    x, w = x.double(), w.double()
    keep = t != ignore
    d = torch.exp(x @ w.T - lse.double()[:, None])
    p = d.clone()
    d[torch.arange(len(t), device=DEV)[keep], t[keep].long()] -= 1
    c = torch.where(keep, gl.double(), 0.0)[:, None]
    return (d * c) @ w, (d * c).T @ x, d * c, p * c


def check_grad(x, w, t, gl, lse=None):
    if lse is None:
        lse = head.token_loss(x, w, t)[1]
    dx, dw = head.token_loss_grad(x, w, t, lse, gl)
    wx, ww, D, pc = defined_grad(x, w, t, lse, gl)
    dt = x.dtype
    ud = 2.0 ** -21 if dt == torch.float32 else U[dt]  # D is held in 16 bits, of 32-bit operands in two halves
    # exp(l - lse): the logit's error, and that of the difference, the factor log2 e and the exponential
    ep = logit_bound(x, w)[:, None] + 4 * U32 * (lse.double().abs()[:, None] + 30)
    # float16 below its smallest step: 2^-25 of the largest |g| 2^-13
    tiny = 0 if dt == torch.bfloat16 else 2.0 ** -37 * gl.abs().max().double()
    e = D.abs() * ud + pc.abs() * ep + tiny
    n = x.shape[0]
    for got, want, other, err, mag, terms in ((dx, wx, w, e, D.abs(), w.shape[0]), (dw, ww, x, e.T, D.abs().T, n)):
        a = other.double().abs()
        passes = 3 if dt == torch.float32 else 1
        tol = err @ a + (mag @ a) * (U32 * (passes * terms + 16) + (2.0 ** -21 if passes == 3 else 0)) + want.abs() * U[dt]
        tol = tol + (2.0 ** -25 if dt == torch.float16 else 0) + 1e-30
        off = (got.double() - want).abs()
        assert (off <= tol).all(), (off / tol).max().item()
    assert (dx[t == -100] == 0).all()
    return dx, dw


SIZES = [(1, 1, 1), (1, 2, 8), (3, 5, 7), (50, 432, 64), (64, 64, 128), (65, 129, 72), (129, 1731, 136), (200, 4099, 333), (257, 1000, 520), (300, 513, 96)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,width", SIZES)
def test_loss(rows, vocab, width, dtype):
    check_loss(*make(rows, vocab, width, dtype)[:3])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,width", SIZES)
def test_grad(rows, vocab, width, dtype):
    check_grad(*make(rows, vocab, width, dtype, seed=1))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,width", [(1024, 8192, 128), (700, 17000, 64), (2100, 4200, 264)])
def test_larger_tiles(rows, vocab, width, dtype):
    x, w, t, gl = make(rows, vocab, width, dtype, seed=2)
    _, lse = check_loss(x, w, t)
    check_grad(x, w, t, gl, lse)


def test_several_pieces_of_the_vocabulary():
    x, w, t, gl = make(8200, 19001, 64, torch.bfloat16, seed=3)
    check_grad(x, w, t, gl)


def test_pieces_for_many_positions():
    x, w, t, gl = make(40000, 9000, 32, torch.bfloat16, seed=3)
    check_grad(x, w, t, gl)


# whole tiles of 256 and 128 with a few rows, columns or positions behind them, and just past what thin tiles take
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,width", [(2049, 4097, 64), (2112, 4160, 72), (2113, 4161, 64), (1090, 1795, 520)])
def test_remainders(rows, vocab, width, dtype):
    x, w, t, gl = make(rows, vocab, width, dtype, seed=7)
    t[:4] = torch.arange(vocab - 4, vocab, device=DEV)
    _, lse = check_loss(x, w, t)
    check_grad(x, w, t, gl, lse)
    q, s = head.quantize_rows(w)
    assert torch.equal(head.token_scores_int8(x, q, s, out_dtype=torch.float32), defined_scores(x, q, s, torch.float32))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("pad,wpad", [(8, 16), (1, 0), (0, 3), (24, 1)])
def test_strides(pad, wpad, dtype):
    x, w, t, gl = make(70, 300, 80, dtype, pad=pad, wpad=wpad)
    check_loss(x, w, t)
    check_grad(x, w, t, gl)


# few positions of a table that is not read in place otherwise
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,width,wpad", [(1, 4096, 333, 0), (2, 70001, 68, 1), (16, 1731, 129, 2), (17, 257, 1030, 3), (32, 20000, 37, 0), (64, 500, 250, 5),
                                                   (100, 17, 20, 1)])
def test_few_positions(rows, vocab, width, wpad, dtype):
    x, w, t, gl = make(rows, vocab, width, dtype, seed=11, wpad=wpad)
    _, lse = check_loss(x, w, t)
    check_grad(x, w, t, gl, lse)


def test_unaligned_storage():
    for dtype in TYPES:
        x, w, t, gl = make(40, 100, 64, dtype)
        held = torch.zeros(40 * 64 + 1, dtype=dtype, device=DEV)
        moved = held[1:].view(40, 64).copy_(x)
        check_loss(moved, w, t)
        check_grad(moved, w, t, gl)


def test_rows_far_apart():
    # offsets past 2^32 bytes: 1100 rows, 4 MB apart
    held = torch.empty(1100 << 21, dtype=torch.bfloat16, device=DEV)
    x, w, t, gl = make(20, 1100, 64, torch.bfloat16)
    far = held.as_strided((1100, 64), (1 << 21, 1)).copy_(w)
    check_loss(x, far, t)
    check_grad(x, far, t, gl)
    q, s = head.quantize_rows(w)
    far = held.view(torch.int8).as_strided((1100, 64), (1 << 22, 1)).copy_(q)
    assert torch.equal(head.token_scores_int8(x, far, s), head.token_scores_int8(x, q, s))


def test_one_row_of_a_wide_buffer():
    held = torch.randn(2, 1 << 22, device=DEV).bfloat16()
    x, w, t, gl = make(1, 20, 64, torch.bfloat16, ignored=0)
    check_loss(held[:1, :64], w, t)
    check_grad(held[1:, :64], w, t, gl)


def test_int32_targets_and_another_ignored_value():
    x, w, t, gl = make(60, 500, 64, torch.bfloat16, tdtype=torch.int32)
    loss, lse = check_loss(x, w, t)
    t2 = torch.where(t == -100, 7, t.long())
    a = head.token_loss(x, w, t2, ignore_index=7)
    keep = (t != -100) & (t != 7)
    assert torch.equal(a[0][keep], loss[keep]) and (a[0][~keep] == 0).all() and torch.equal(a[1], lse)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_all_positions_ignored(dtype):
    x, w, t, gl = make(33, 70, 40, dtype)
    t.fill_(-100)
    loss, lse = check_loss(x, w, t)
    dx, dw = head.token_loss_grad(x, w, t, lse, gl)
    assert (dx == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf")])
def test_padding_may_hold_anything(dtype, junk):
    x, w, t, gl = make(90, 400, 72, dtype)
    keep = t != -100
    loss, lse = head.token_loss(x, w, t)
    dx, dw = head.token_loss_grad(x, w, t, lse, gl)
    x2, gl2, lse2 = x.clone(), gl.clone(), lse.clone()
    x2[~keep], gl2[~keep], lse2[~keep] = junk, junk, junk
    loss2, got = head.token_loss(x2, w, t)
    assert torch.equal(loss2, loss) and torch.equal(got[keep], lse[keep])
    dx2, dw2 = head.token_loss_grad(x2, w, t, lse2, gl2)
    # (the scale of the logits' gradient is that of the counted positions alone)
    assert torch.equal(dx2, dx) and torch.equal(dw2, dw)


def test_targets_out_of_range_are_loud():
    x, w, t, gl = make(30, 50, 64, torch.bfloat16, ignored=0)
    t[3], t[4] = 50, -1
    loss, lse = head.token_loss(x, w, t)
    bad = torch.zeros(30, dtype=torch.bool, device=DEV)
    bad[3:5] = True
    assert loss[bad].isnan().all() and not loss[~bad].isnan().any() and not lse.isnan().any()
    dx, dw = head.token_loss_grad(x, w, t, lse, gl)
    assert dx[bad].isnan().all() and not dx[~bad].isnan().any() and dw.isnan().all()


def test_infinite_and_not_a_number():
    x, w, t, _ = make(10, 40, 64, torch.bfloat16, ignored=0)
    x[2, 5], x[7, 1] = float("nan"), float("inf")
    loss, lse = head.token_loss(x, w, t)
    ok = torch.ones(10, dtype=torch.bool, device=DEV)
    ok[2] = ok[7] = False
    assert not torch.isfinite(loss[~ok]).any()
    good = head.token_loss(x[ok].contiguous(), w, t[ok])
    assert torch.equal(loss[ok], good[0]) and torch.equal(lse[ok], good[1])


@pytest.mark.parametrize("scale", [1e-30, 1e-4, 1e4])
def test_32_bit_ranges(scale):
    # the split halves follow the tensor's largest value: products of very small and very large tensors
    for rows, vocab, width in ((40, 300, 96), (1100, 2100, 160)):
        x, w, t, gl = make(rows, vocab, width, torch.float32)
        check_loss(x * scale, w / scale, t)
        check_grad(x * scale, w / scale, t, gl)


def test_large_logits():
    for dtype in TYPES:
        x, w, t, gl = make(50, 600, 64, dtype)
        _, lse = check_loss(x * 64, w, t)
        check_grad(x * 64, w, t, gl, lse)


def test_small_gradients_in_float16():
    x, w, t, gl = make(64, 4096, 64, torch.float16)
    check_grad(x, w, t, gl * 2.0 ** -8)
    dx, dw = check_grad(x, w, t, gl * 2.0 ** 10)
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()


def test_one_gradient_alone():
    x, w, t, gl = make(70, 500, 72, torch.bfloat16)
    lse = head.token_loss(x, w, t)[1]
    dx, dw = head.token_loss_grad(x, w, t, lse, gl)
    a, none = head.token_loss_grad(x, w, t, lse, gl, need_weight=False)
    assert none is None and torch.equal(a, dx)
    none, b = head.token_loss_grad(x, w, t, lse, gl, need_hidden=False)
    assert none is None and torch.equal(b, dw)


def test_no_positions():
    x, w, t, gl = make(0, 30, 64, torch.float32)
    loss, lse = head.token_loss(x, w, t)
    assert loss.shape == lse.shape == (0,)
    for dtype in TYPES:
        dx, dw = head.token_loss_grad(x.to(dtype), w.to(dtype), t, lse, gl)
        assert dx.shape == (0, 64) and (dw == 0).all() and dw.shape == w.shape
    q, s = head.quantize_rows(w)
    assert head.token_scores_int8(x, q, s).shape == (0, 30)
    assert head.quantize_rows(x)[0].shape == (0, 64)


def test_gradient_against_differences():
    x, w, t, gl = make(12, 30, 16, torch.float32, seed=4)
    loss, lse = head.token_loss(x, w, t)
    dx, dw = head.token_loss_grad(x, w, t, lse, gl)
    f = lambda a, b: (defined_loss(a, b, t)[0] * gl.double()).sum()  # noqa: E731
    h = 2.0 ** -12  # the third derivative's term is below 1e-7 for these values
    for m, d, k in ((x, dx, 0), (w, dw, 1)):
        for i, j in ((0, 0), (3, 5), (11, 15), (7, 9)):
            e = torch.zeros_like(m, dtype=torch.float64)
            e[i, j] = h
            a = (m.double() + e, w.double()) if k == 0 else (x.double(), m.double() + e)
            b = (m.double() - e, w.double()) if k == 0 else (x.double(), m.double() - e)
            assert abs(((f(*a) - f(*b)) / (2 * h)).item() - d[i, j].item()) < 1e-5


def defined_scores(x, q, s, out):
    h = x.float()
    sx = h.abs().amax(1) * torch.tensor(1 / 127, device=DEV, dtype=torch.float32)
    c = torch.round(h / torch.where(sx > 0, sx, 1.0)[:, None])
    return ((c.double() @ q.double().T).float() * sx[:, None] * s).to(out)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("out", TYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,width", SIZES + [(1, 4096, 512), (16, 5000, 1024), (17, 5001, 700), (33, 333, 2048)])
def test_scores(rows, vocab, width, dtype, out):
    x, w, _, _ = make(rows, vocab, width, dtype, seed=5)
    q, s = head.quantize_rows(w)
    sw = w.float().abs().amax(1) * torch.tensor(1 / 127, device=DEV, dtype=torch.float32)
    assert torch.equal(s, sw)
    assert torch.equal(q, torch.round(w.float() / torch.where(sw > 0, sw, 1.0)[:, None]).to(torch.int8))
    got = head.token_scores_int8(x, q, s, out_dtype=out)
    # integers are exact and the two products are rounded alike
    assert got.dtype == out and torch.equal(got, defined_scores(x, q, s, out))


@pytest.mark.parametrize("rows,vocab,width", [(2000, 8192, 256), (600, 17000, 96), (2050, 4100, 1000)])
def test_scores_larger(rows, vocab, width):
    x, w, _, _ = make(rows, vocab, width, torch.float16, seed=6, pad=3)
    q, s = head.quantize_rows(w)
    assert torch.equal(head.token_scores_int8(x, q, s, out_dtype=torch.float32), defined_scores(x, q, s, torch.float32))


def test_scores_of_padded_weights_and_odd_rows():
    x, w, _, _ = make(9, 200, 100, torch.bfloat16)
    q, s = head.quantize_rows(w)
    for extra in (1, 4, 12, 28):
        held = torch.full((200, 100 + extra), 111, dtype=torch.int8, device=DEV)
        held[:, :100] = q
        assert torch.equal(head.token_scores_int8(x, held[:, :100], s), head.token_scores_int8(x, q, s))


def test_scores_of_zeros_and_of_junk():
    x, w, _, _ = make(5, 60, 64, torch.float32)
    x[1], x[3, 2], x[4, 0] = 0, float("nan"), float("inf")
    w[7] = 0
    q, s = head.quantize_rows(w)
    got = head.token_scores_int8(x, q, s)
    assert (got[1] == 0).all() and got[3].isnan().all() and got[4].isnan().all() and (got[[0, 2], 7] == 0).all()
    assert torch.isfinite(got[[0, 2]]).all()


def test_scores_near_the_integers_limit():
    x, w = torch.ones(3, 131072, device=DEV), torch.ones(5, 131072, device=DEV)
    q, s = head.quantize_rows(w)
    assert (q == 127).all()
    got = head.token_scores_int8(x, q, s)
    assert torch.equal(got, defined_scores(x, q, s, torch.float32)) and abs(got[0, 0].item() / 131072 - 1) < 1e-5


def test_output_rows_behind_the_last_column_stay():
    x, w, _, _ = make(6, 70, 64, torch.bfloat16)
    q, s = head.quantize_rows(w)
    want = head.token_scores_int8(x, q, s, out_dtype=torch.float32)
    for ldo in (70, 71, 72, 128):  # aligned and unaligned row strides of a caller's buffer
        held = torch.full((7, ldo), 5.0, device=DEV)
        L = _native.lib()
        n = L.pst_token_scores_i8_workspace(1, x.data_ptr(), 64, q.data_ptr(), 64, 6, 70, 64)
        ws = torch.empty(n + 256, dtype=torch.uint8, device=DEV)
        assert L.pst_token_scores_i8(0, 1, x.data_ptr(), 64, q.data_ptr(), 64, s.data_ptr(), 6, 70, 64, 0, held.data_ptr(), ldo,
                                     (ws.data_ptr() + 255) // 256 * 256, n, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(held[:6, :70], want) and (held[:6, 70:] == 5).all() and (held[6] == 5).all()


def test_same_bits_each_time():
    x, w, t, gl = make(1000, 4099, 200, torch.bfloat16)
    first = None
    for _ in range(3):
        loss, lse = head.token_loss(x, w, t)
        got = (loss, lse) + head.token_loss_grad(x, w, t, lse, gl)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def step(x, w, t, gl, q, s):
    loss, lse = head.token_loss(x, w, t)
    dx, dw = head.token_loss_grad(x, w, t, lse, gl)
    return loss, lse, dx, dw, head.token_scores_int8(x, q, s, out_dtype=torch.float32)


def test_captured_and_replayed():
    """Graphs and eager calls of other sizes between their replays: each has its own workspace."""
    sets, graphs, outs = [], [], []
    for k, (rows, vocab) in enumerate(((100, 700), (64, 1500), (2048, 8200), (1100, 4099))):
        x, w, t, gl = make(rows, vocab, 136, (torch.float32, torch.bfloat16, torch.bfloat16, torch.float32)[k], seed=k)
        sets.append((x, w, t, gl) + head.quantize_rows(w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a in sets:
            step(*a)
    torch.cuda.current_stream().wait_stream(side)
    for a in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*a))
        graphs.append(g)
    for seed in range(3):
        for k, a in enumerate(sets):
            fresh = make(a[0].shape[0], a[1].shape[0], 136, a[0].dtype, seed=10 + seed)
            for to, frm in zip(a[:4], fresh):
                to.copy_(frm)
            fq = head.quantize_rows(a[1])
            a[4].copy_(fq[0]), a[5].copy_(fq[1])
        for g in graphs:
            g.replay()
        want = [step(*a) for a in sets]
        torch.cuda.synchronize()
        for o, e in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(o, e))


def test_another_stream():
    x, w, t, gl = make(300, 3000, 128, torch.bfloat16)
    q, s = head.quantize_rows(w)
    want = step(x, w, t, gl, q, s)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append(step(x, w, t, gl, q, s))
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_used_together():
    """A table trained on the ids by plain gradient steps, then served in 8 bits."""
    x, w, t, _ = make(256, 432, 64, torch.float32, seed=8, ignored=0.1)
    keep = t != -100
    gl = keep.float() / keep.sum()
    for _ in range(5):
        loss, lse = head.token_loss(x, w, t)
        dx, dw = head.token_loss_grad(x, w, t, lse, gl)
        wx, ww, _, _ = defined_grad(x, w, t, lse, gl)
        assert (dw.double() - ww).norm() <= 1e-5 * ww.norm() and (dx.double() - wx).norm() <= 1e-5 * wx.norm()
        w -= 0.5 * dw
    q, s = head.quantize_rows(w)
    scores = head.token_scores_int8(x, q, s)
    # each product is off by half a step of either factor's 127 steps
    full = x.double() @ w.double().T
    tol = 0.5 / 127 * (x.double().abs().amax(1)[:, None] * w.double().abs().sum(1) + x.double().abs().sum(1)[:, None] * w.double().abs().amax(1)) * 1.02
    assert ((scores.double() - full).abs() <= tol).all()


def test_refusals_on_the_gpu():
    x, w, t, gl = make(8, 30, 64, torch.bfloat16)
    lse = torch.zeros(8, device=DEV)
    q, s = head.quantize_rows(w)
    with pytest.raises(ValueError, match="one type"):
        head.token_loss(x, w.float(), t)
    with pytest.raises(ValueError, match="columns"):
        head.token_loss(x, w[:, :32], t)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        head.token_loss(x.double(), w.double(), t)
    with pytest.raises(ValueError, match="int64 or int32"):
        head.token_loss(x, w, t.float())
    with pytest.raises(ValueError, match="vector of 8"):
        head.token_loss(x, w, t[:7])
    with pytest.raises(ValueError, match="is on cpu"):
        head.token_loss(x, w.cpu(), t)
    with pytest.raises(ValueError, match="column stride"):
        head.token_loss(x.t(), w, t)
    with pytest.raises(ValueError, match="float32 is needed"):
        head.token_loss_grad(x, w, t, lse.double(), gl)
    with pytest.raises(ValueError, match="int8"):
        head.token_scores_int8(x, w, s)
    with pytest.raises(ValueError, match="vector of 30"):
        head.token_scores_int8(x, q, s[:29])
    with pytest.raises(ValueError, match="out_dtype"):
        head.token_scores_int8(x, q, s, out_dtype=torch.float64)


class TokenLoss(torch.autograd.Function):
    """The operators under autograd, as the integration notes give them."""

    @staticmethod
    def forward(ctx, hidden, weight, targets):
        loss, lse = head.token_loss(hidden, weight, targets)
        ctx.save_for_backward(hidden, weight, targets, lse)
        return loss

    @staticmethod
    def backward(ctx, grad_loss):
        hidden, weight, targets, lse = ctx.saved_tensors
        return (*head.token_loss_grad(hidden, weight, targets, lse, grad_loss.contiguous()), None)


def test_under_autograd():
    x, w, t, _ = make(60, 432, 48, torch.float32, seed=9)
    x.requires_grad_(), w.requires_grad_()
    n = (t != -100).sum()
    TokenLoss.apply(x, w, t).sum().div(n).backward()
    a, b = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    torch.nn.functional.cross_entropy(a @ b.T, t, ignore_index=-100).backward()
    # 60 and 432 terms, split products of 2^-21, exponents off by a few of 2^-24: far below 1e-5 of the norm
    assert (x.grad.double() - a.grad).norm() <= 1e-5 * a.grad.norm()
    assert (w.grad.double() - b.grad).norm() <= 1e-5 * b.grad.norm()


@pytest.mark.parametrize("rows,vocab,width", [(90, 400, 72), (300, 4099, 333), (1100, 2100, 160)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_padding_may_hold_large_numbers(rows, vocab, width, dtype):
    x, w, t, gl = make(rows, vocab, width, dtype)
    keep = t != -100
    loss, lse = head.token_loss(x, w, t)
    dx, dw = head.token_loss_grad(x, w, t, lse, gl)
    x2 = x.clone()
    x2[~keep] = 1e30
    loss2, lse2 = head.token_loss(x2, w, t)
    assert torch.equal(loss2, loss) and torch.equal(lse2[keep], lse[keep])
    dx2, dw2 = head.token_loss_grad(x2, w, t, lse2, gl)
    assert torch.equal(dx2, dx) and torch.equal(dw2, dw)


@pytest.mark.parametrize("rows,vocab,width", [(300, 4099, 333), (1100, 2100, 160)])
def test_32_bit_positions_of_very_different_sizes(rows, vocab, width):
    # each position's loss and lse within the bound of its own values (ignored ones' lse too), whatever the others hold
    x, w, t, _ = make(rows, vocab, width, torch.float32)
    scale = 10.0 ** torch.linspace(-2, 16, rows, device=DEV)
    check_loss(x * scale[:, None], w, t)


@pytest.mark.parametrize("dtype,scale", [(torch.bfloat16, 1e15), (torch.bfloat16, 1e30), (torch.float16, 1e4), (torch.float32, 1e30)])
def test_logits_of_any_finite_size(dtype, scale):
    for rows, vocab, width in ((40, 300, 96), (300, 4099, 333)):
        x, w, t, _ = make(rows, vocab, width, torch.float32)
        check_loss((x * scale / 8).to(dtype), w.to(dtype), t)
