"""Token head: operators over a learned table `weight` [V, d] with one row per token id, for sequence models over the
ids that the tokenizer makes (`include/pst.h`, section "Token head"; `Tokenizer.codebook_aux` gives the same kind of
scores over the implicit codebook).

    loss, lse = token_loss(hidden, weight, targets)              # softmax cross entropy per position, no logits kept
    loss.sum().backward()                                        # where hidden or weight requires grad, or by hand:
    dhidden, dweight = token_loss_grad(hidden, weight, targets, lse, grad_loss)
    qweight, scale = quantize_rows(weight)                       # once
    scores = token_scores_int8(hidden, qweight, scale)           # 8-bit products, a scale for each row and each id

Arguments are torch tensors on one GPU: matrices with unit column stride and any row stride (rows more than
2^21 elements apart, 2^23 of an int8 table, are copied together first). Calls launch on torch's
current stream of that GPU and do not synchronise; workspaces come from torch's allocator, so calls on several streams
and captured graphs each have their own. Types: float32, bfloat16, float16 (hidden and weight of the same type).
`ValueError` names an argument that does not fit, `NotImplementedError` a size past the limits (2^30 rows or ids,
2^20 columns, 131072 of 8-bit scores), `PstError` what the runtime reported. torch has to be imported before
pst_amd loads libpst, so that both use one HIP runtime.
"""
import functools

from . import _native

_TYPES = {"torch.float32": 0, "torch.bfloat16": 1, "torch.float16": 2}  # PST_F32, PST_BF16, PST_F16
_target_bits = {}  # torch.dtype -> bits
_type_of = {}  # torch.dtype -> code, filled on first use (a dtype's text costs more to make than to look up)


def _code(t, name):
    d = t.dtype
    if d not in _type_of:
        if str(d) not in _TYPES:
            raise ValueError(f"{name} is {d}: float32, bfloat16 or float16 is needed")
        _type_of[d] = _TYPES[str(d)]
    return _type_of[d]


_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch
        _native.lib()
        if not _native.shares_torch_runtime:
            raise _native.PstError("import torch before pst_amd loads libpst: the two hold different HIP runtimes")
        for bits in (32, 64):
            _target_bits[getattr(torch, f"int{bits}")] = bits
        _torch_module = torch  # last: another thread that sees it goes on with what is above
    return _torch_module


def _check(rc):
    if rc != _native.PST_OK:
        _native.raise_for(rc, _native.lib().pst_head_error().decode())


def _device(t, name):
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}: a GPU tensor is needed")
    return t.device


def _matrix(t, name, device=None):
    """(pointer, row stride) of a matrix with unit column stride."""
    if t.dim() != 2:
        raise ValueError(f"{name} has {t.dim()} dimensions: 2 are needed")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}: {device} is needed")
    rows, cols = t.shape
    s0, s1 = t.stride()
    if cols > 1 and s1 != 1:
        raise ValueError(f"{name} has a column stride of {s1}: 1 is needed")
    if rows <= 1:
        s0 = cols
    elif s0 < cols:
        raise ValueError(f"{name} has overlapping rows (row stride {s0} of {cols} columns)")
    return t.data_ptr(), s0


_FAR, _FAR_INT8 = 1 << 21, 1 << 23  # row strides, in elements, that the kernels' offsets within a tile take


def _near(t, name, device=None, far=_FAR):
    """(matrix, pointer, row stride), a copy where the rows are further apart than `far`."""
    p, ld = _matrix(t, name, device)
    if ld > far:
        t = t.contiguous()
        p, ld = _matrix(t, name, device)
    return t, p, ld


def _vector(t, name, n, device, dtype=None):
    if t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} has shape {tuple(t.shape)} and strides {t.stride()}: a contiguous vector of {n} is needed")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}: {device} is needed")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} is {t.dtype}: {dtype} is needed")
    return t.data_ptr()


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(fn, *key):
    n = getattr(_native.lib(), fn)(*key)
    _check(min(n, 0))
    return n


def _workspace(torch, device, fn, ctype, x, ldx, w, ldw, rows, vocab, width):
    """A call's workspace (torch's allocations are aligned to 512 bytes) and its size."""
    # a pointer counts by its alignment alone
    n = _workspace_bytes(fn, ctype, 256 + (x & 15), ldx, 256 + (w & 15), ldw, rows, vocab, width)
    return torch.empty(n, dtype=torch.uint8, device=device), n


def _stream(torch, device):
    return torch._C._cuda_getCurrentRawStream(device.index)  # torch.cuda.current_stream without the object


def _head(torch, hidden, weight):
    device = _device(hidden, "hidden")
    code = _code(hidden, "hidden")
    if weight.dtype != hidden.dtype:
        raise ValueError(f"weight is {weight.dtype} and hidden {hidden.dtype}: one type is needed")
    hidden, x, ldx = _near(hidden, "hidden")
    weight, w, ldw = _near(weight, "weight", device)
    if weight.shape[1] != hidden.shape[1]:
        raise ValueError(f"weight has {weight.shape[1]} columns and hidden {hidden.shape[1]}")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight has shape {tuple(weight.shape)}: a row and a column are needed at least")
    return hidden, weight, device, code, x, ldx, w, ldw


def _targets(targets, rows, device):
    bits = _target_bits.get(targets.dtype)
    if bits is None:
        raise ValueError(f"targets are {targets.dtype}: int64 or int32 is needed")
    return _vector(targets, "targets", rows, device), bits


_function = None


def _differentiable(torch):
    """token_loss as an autograd function, made on first use."""
    global _function
    if _function is None:
        class TokenLoss(torch.autograd.Function):
            @staticmethod
            def forward(ctx, hidden, weight, targets, ignore_index):
                loss, lse = _loss(torch, hidden, weight, targets, ignore_index)
                ctx.save_for_backward(hidden, weight, targets, lse)
                ctx.ignore_index = ignore_index
                ctx.set_materialize_grads(False)
                return loss, lse

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, grad_loss, grad_lse):
                if grad_lse is not None:
                    raise NotImplementedError("lse of token_loss has no gradient: use loss, or lse.detach()")
                if grad_loss is None:
                    return None, None, None, None
                hidden, weight, targets, lse = ctx.saved_tensors
                need_hidden, need_weight = ctx.needs_input_grad[:2]
                return (*token_loss_grad(hidden, weight, targets, lse, grad_loss.contiguous(), ignore_index=ctx.ignore_index,
                                         need_hidden=need_hidden, need_weight=need_weight), None, None)

        _function = TokenLoss
    return _function


def token_loss(hidden, weight, targets, *, ignore_index=-100):
    """Softmax cross entropy of each position over the vocabulary: (loss [N], lse [N]) in float32,
    lse[n] = log sum_v exp(<hidden[n], weight[v]>), loss[n] = lse[n] - <hidden[n], weight[targets[n]]>.

    `hidden` [N, d], `weight` [V, d], `targets` [N] int64 or int32. Positions whose target is `ignore_index` have loss
    0; a target outside [0, V) that is not `ignore_index` gives loss NaN. `lse` is what `token_loss_grad` takes.

    Where grad mode is on and `hidden` or `weight` requires grad, `loss` is differentiable (once) by `token_loss_grad`; a
    gradient that arrives at `lse` raises `NotImplementedError`."""
    torch = _torch()
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _differentiable(torch).apply(hidden, weight, targets, ignore_index)
    return _loss(torch, hidden, weight, targets, ignore_index)


def _loss(torch, hidden, weight, targets, ignore_index):
    hidden, weight, device, code, x, ldx, w, ldw = _head(torch, hidden, weight)
    rows, width = hidden.shape
    vocab = weight.shape[0]
    t, bits = _targets(targets, rows, device)
    loss = torch.empty(rows, dtype=torch.float32, device=device)
    lse = torch.empty(rows, dtype=torch.float32, device=device)
    if rows:
        ws, wn = _workspace(torch, device, "pst_token_loss_workspace", code, x, ldx, w, ldw, rows, vocab, width)
        _check(_native.lib().pst_token_loss(device.index, code, x, ldx, w, ldw, rows, vocab, width, t, bits, ignore_index,
                                            loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), wn, _stream(torch, device)))
    return loss, lse


def token_loss_grad(hidden, weight, targets, lse, grad_loss, *, ignore_index=-100, need_hidden=True, need_weight=True):
    """Gradients of sum_n grad_loss[n] loss[n]: (for hidden, for weight), of their type; None where not needed. They are
    detached: what autograd has for `token_loss`, called by hand.

    `lse` [N] float32 from `token_loss`, `grad_loss` [N] float32. Positions whose target is `ignore_index` have zero
    gradient and add nothing to the weight's, whatever their hidden row holds; a target out of range gives NaN. The logits' gradient is held to 2^-16 of each entry for 16-bit types.
    float16: scale the loss, since gradients below 6e-8 vanish in the type."""
    torch = _torch()
    hidden, weight, device, code, x, ldx, w, ldw = _head(torch, hidden, weight)
    rows, width = hidden.shape
    vocab = weight.shape[0]
    t, bits = _targets(targets, rows, device)
    sp = _vector(lse, "lse", rows, device, torch.float32)
    gp = _vector(grad_loss, "grad_loss", rows, device, torch.float32)
    dx = torch.empty((rows, width), dtype=hidden.dtype, device=device) if need_hidden else None
    dw = torch.empty((vocab, width), dtype=weight.dtype, device=device) if need_weight else None
    if dw is not None or (dx is not None and rows):
        ws, wn = _workspace(torch, device, "pst_token_loss_grad_workspace", code, x, ldx, w, ldw, rows, vocab, width)
        _check(_native.lib().pst_token_loss_grad(
            device.index, code, x, ldx, w, ldw, rows, vocab, width, t, bits, ignore_index, sp, gp,
            dx.data_ptr() if dx is not None else None, width, dw.data_ptr() if dw is not None else None, width, ws.data_ptr(), wn,
            _stream(torch, device)))
    return dx, dw


def quantize_rows(x):
    """(int8 [R, d], float32 scale [R]): scale = max |row| * (1/127), values rint(x / scale). A row of zeros has scale 0;
    one that holds an infinity or NaN has scale NaN and values 0."""
    torch = _torch()
    device = _device(x, "x")
    code = _code(x, "x")
    p, ld = _matrix(x, "x")
    rows, width = x.shape
    if width < 1:
        raise ValueError(f"x has shape {tuple(x.shape)}: a column is needed at least")
    q = torch.empty((rows, width), dtype=torch.int8, device=device)
    scale = torch.empty(rows, dtype=torch.float32, device=device)
    if rows:
        _check(_native.lib().pst_quantize_rows(device.index, code, p, ld, rows, width, q.data_ptr(), width, scale.data_ptr(),
                                               _stream(torch, device)))
    return q, scale


def token_scores_int8(hidden, qweight, scale, *, out_dtype=None):
    """Scores [N, V] of all token ids in 8-bit products: hidden's rows are rounded to 8 bits with a scale each
    (`quantize_rows`' rule) within the call, `qweight` int8 [V, d] and `scale` float32 [V] are `quantize_rows` of the
    table. Sums are exact. `out_dtype`: float32, bfloat16 or float16, hidden's by default. The result's rows are
    aligned: its row stride is V rounded up to a multiple of 64. They are detached: rounding has no gradient."""
    torch = _torch()
    device = _device(hidden, "hidden")
    code = _code(hidden, "hidden")
    x, ldx = _matrix(hidden, "hidden")
    rows, width = hidden.shape
    if qweight.dtype != torch.int8:
        raise ValueError(f"qweight is {qweight.dtype}: int8 is needed")
    qweight, w, ldw = _near(qweight, "qweight", device, _FAR_INT8)
    vocab = qweight.shape[0]
    if qweight.shape[1] != width:
        raise ValueError(f"qweight has {qweight.shape[1]} columns and hidden {width}")
    if vocab < 1 or width < 1:
        raise ValueError(f"qweight has shape {tuple(qweight.shape)}: a row and a column are needed at least")
    sp = _vector(scale, "scale", vocab, device, torch.float32)
    ldo = (vocab + 63) // 64 * 64
    held = torch.empty((rows, ldo), dtype=out_dtype or hidden.dtype, device=device)
    out_code = _code(held, "out_dtype")
    out = held[:, :vocab]
    if rows:
        ws, wn = _workspace(torch, device, "pst_token_scores_i8_workspace", code, x, ldx, w, ldw, rows, vocab, width)
        _check(_native.lib().pst_token_scores_i8(device.index, code, x, ldx, w, ldw, sp, rows, vocab, width, out_code,
                                                 out.data_ptr(), ldo, ws.data_ptr(), wn, _stream(torch, device)))
    return out
