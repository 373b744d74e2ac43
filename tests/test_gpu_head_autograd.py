"""The token head's loss under torch's autograd: the gradients are token_loss_grad's, of the sides that need one, and none is
lost without a word."""
import pytest
import torch  # before libpst loads: one HIP runtime serves both

from pst_amd import head

pytestmark = pytest.mark.gpu

DEV = "cuda"


def make(rows=60, vocab=432, width=48, dtype=torch.float32, seed=0, ignore=-100):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, width, generator=g, device=DEV).to(dtype)
    w = (torch.randn(vocab, width, generator=g, device=DEV) * width ** -0.5).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    t[torch.rand(rows, generator=g, device=DEV) < 0.2] = ignore
    return x, w, t


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("sides", [(True, True), (True, False), (False, True)], ids=str)
def test_gradients_are_those_by_hand(dtype, sides):
    x, w, t = make(dtype=dtype)
    want_loss, want_lse = head.token_loss(x, w, t)
    n = (t != -100).sum()
    gl = torch.full((len(t),), 1.0, device=DEV) / n
    want = head.token_loss_grad(x, w, t, want_lse, gl)
    x.requires_grad_(sides[0]), w.requires_grad_(sides[1])
    loss, lse = head.token_loss(x, w, t)
    assert loss.requires_grad and torch.equal(loss, want_loss) and torch.equal(lse, want_lse)
    (loss.sum() / n).backward()  # (an expanded gradient of the loss)
    for m, d, need in zip((x, w), want, sides):
        assert torch.equal(m.grad, d) if need else m.grad is None


def test_another_term_keeps_its_gradient_beside_it():
    x, w, t = make()
    x.requires_grad_()
    loss, lse = head.token_loss(x, w, t)
    gl = torch.linspace(0.5, 1.5, len(t), device=DEV)
    ((loss * gl).sum() + (x * 3).sum()).backward()
    dx, _ = head.token_loss_grad(x, w, t, lse, gl)
    assert torch.equal(x.grad, dx + 3)


def test_another_ignored_value():
    x, w, t = make(ignore=7)
    x.requires_grad_()
    loss, lse = head.token_loss(x, w, t, ignore_index=7)
    loss.sum().backward()
    assert (x.grad[t == 7] == 0).all() and (x.grad[t != 7] != 0).any(1).all()


def test_without_grad_mode_nothing_is_recorded():
    x, w, t = make()
    x.requires_grad_()
    with torch.no_grad():
        loss, lse = head.token_loss(x, w, t)
    assert not loss.requires_grad and not lse.requires_grad
    loss, _ = head.token_loss(x.detach(), w, t)
    assert not loss.requires_grad


def test_a_gradient_for_lse_is_refused():
    x, w, t = make()
    x.requires_grad_()
    loss, lse = head.token_loss(x, w, t)
    with pytest.raises(NotImplementedError, match="lse"):
        (loss.sum() + (lse * lse).sum()).backward()
    loss, lse = head.token_loss(x, w, t)
    (loss.sum() + (lse.detach() ** 2).sum()).backward()


def test_second_derivatives_are_refused():
    x, w, t = make()
    x.requires_grad_()
    loss, _ = head.token_loss(x, w, t)
    d, = torch.autograd.grad((loss * loss).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


def test_inside_a_function_of_the_caller_s():
    class Mine(torch.autograd.Function):
        @staticmethod
        def forward(ctx, hidden, weight, targets):
            loss, lse = head.token_loss(hidden, weight, targets)
            ctx.save_for_backward(hidden, weight, targets, lse)
            return loss

        @staticmethod
        def backward(ctx, g):
            return (*head.token_loss_grad(*ctx.saved_tensors, g.contiguous()), None)

    x, w, t = make()
    x.requires_grad_(), w.requires_grad_()
    a = torch.autograd.grad(Mine.apply(x, w, t).sum(), (x, w))
    b = torch.autograd.grad(head.token_loss(x, w, t)[0].sum(), (x, w))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_captured_and_replayed():
    x, w, t = make(300, 1500, 72, torch.bfloat16)
    x.requires_grad_(), w.requires_grad_()

    def step():
        loss, _ = head.token_loss(x, w, t)
        return (loss.detach(), *torch.autograd.grad(loss.mean(), (x, w)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # (its graph is gone when it returns)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2, 3):
        fresh = make(300, 1500, 72, torch.bfloat16, seed=seed)
        with torch.no_grad():
            for to, frm in zip((x, w, t), fresh):
                to.copy_(frm)
        graph.replay()
        a, b = x.detach(), w.detach()
        loss, lse = head.token_loss(a, b, t)
        want = (loss, *head.token_loss_grad(a, b, t, lse, torch.full_like(loss, 1 / len(t))))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_rows_further_apart_than_the_kernels_take():
    """The last positions of whole sequences, and tables that are slices of something wide: strides past 2^21 (int8 2^23)."""
    states = torch.zeros(5, 4096, 1024, dtype=torch.bfloat16, device=DEV)
    x, w, t = make(5, 40, 1024, torch.bfloat16)
    states[:, -1] = x
    far = states[:, -1]
    assert far.stride(0) == 1 << 22
    wide = torch.zeros(40, (1 << 21) + 8, dtype=torch.bfloat16, device=DEV)
    wide[:, :1024] = w
    loss, lse = head.token_loss(x, w, t)
    gl = torch.ones_like(loss)
    dx, dw = head.token_loss_grad(x, w, t, lse, gl)
    for a, b in ((far, w), (x, wide[:, :1024]), (far, wide[:, :1024])):
        got, got_lse = head.token_loss(a, b, t)
        assert torch.equal(got, loss) and torch.equal(got_lse, lse)
        assert all(torch.equal(p, q) for p, q in zip(head.token_loss_grad(a, b, t, lse, gl), (dx, dw)))
    a = far.detach().requires_grad_()
    head.token_loss(a, w, t)[0].sum().backward()
    assert torch.equal(a.grad, dx)
    q, s = head.quantize_rows(w)
    fq, fs = head.quantize_rows(wide[:, :1024])
    assert torch.equal(fq, q) and torch.equal(fs, s)
    want = head.token_scores_int8(x, q, s)
    held = torch.zeros(40, (1 << 23) + 16, dtype=torch.int8, device=DEV)
    held[:, :1024] = q
    for table in (q, held[:, :1024]):
        assert torch.equal(head.token_scores_int8(far, table, s), want)
