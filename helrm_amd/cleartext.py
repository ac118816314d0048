"""Operators that train and score a model in the clear, on torch tensors.

The encrypted path (`orion_host`) evaluates a model that was trained: its
table, its Linears, its degree-3 activations.  These are the operators of
that training and of scoring beside it, on the same card:

    layer_norm      y = (x - mean) / sqrt(var + eps) * weight + bias
    gated_mlp       y = (act(x gate^T) * (x up^T)) down^T
    cross_entropy   log sum_v exp <x, table[v]> - <x, table[target]>

Each has a `_forward` and a `_backward` call, which a training loop of one's
own makes, and a form for torch's autograd.  The matrices' last dimension is
the vector; leading dimensions are rows.  Types: float32, bfloat16, float16,
one for all of an operator's tensors (a norm's weight and bias may be float32
beside any); sums and softmax statistics are float32.  Tensors of the same rows
have the same leading dimensions, or the rows in one.

Work goes to torch's current stream of the tensors' device and nothing waits
for it.  Outputs and workspaces come from torch's allocator; a tensor that
another stream made or still writes has to be waited for by the caller, as
with torch's own operators.  A layout that the kernels do not take (a last
dimension that is not contiguous, rows that overlap) is copied first.
Shapes and types that do not fit raise ValueError, tensors with a forward-mode
tangent NotImplementedError; HipError holds what the library refuses.
"""
import ctypes

import torch
from torch.autograd import forward_ad

from .backend import CrossEntropyArgs, GatedMLPArgs, HipError, LayerNormArgs, LossTotalArgs, load_library

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTS = {"silu": 0, "gelu": 1}

# the handle of the current stream, without making a Stream object of it (a microsecond of a small call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


# entry point -> (the call, its workspace's size or None), once the library is there
_calls = {}


def _library():
    lib = load_library()
    # a stream or pointer of one HIP runtime means nothing to another one: torch brings its own, and the
    # library takes that one if it is there when the library is loaded
    with open("/proc/self/maps") as f:
        runtimes = {line.split()[-1] for line in f if "libamdhip64.so" in line}
    if len(runtimes) > 1:
        raise HipError("two HIP runtimes in one process (" + ", ".join(sorted(runtimes))
                       + "): import torch before the library is loaded")
    calls = {}
    for name in ("LayerNorm", "LayerNormGrad", "GatedMLP", "GatedMLPGrad", "CrossEntropy", "CrossEntropyGrad", "LossTotal"):
        call, size = getattr(lib, name), getattr(lib, name + "Workspace") if name != "LayerNorm" else None
        call.argtypes, call.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
        if size is not None:
            size.argtypes, size.restype = [ctypes.c_void_p], ctypes.c_long
        calls[name] = call, size
    _calls.update(calls)   # all at once: another thread finds none of them or every one


def _refused():
    raise HipError(load_library().GetLastError().decode())


def _call(name, args, device):
    """Queue one entry point on the current stream; a workspace of the size it asks for is there while it runs."""
    if not _calls:
        _library()
    call, size = _calls[name]
    index = device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _call(name, args, device)
    ref = ctypes.byref(args)
    space = None
    if size is not None and not args.workspace:
        need = size(ref)
        if need < 0:
            _refused()
        space = torch.empty(need, dtype=torch.uint8, device=device)
        args.workspace, args.workspaceBytes = space.data_ptr(), need
    if call(ref, _raw_stream(index)):
        _refused()


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _sized(n, name):
    # (a C int takes a larger size modulo 2^32, without an error)
    if n >= 1 << 31:
        raise ValueError(f"{name}: {n}, the most is 2^31 - 1")


def _no_tangent(t, name):
    # (a kernel reads the storage, where a dual tensor's tangent is not: it would be lost without a word)
    if forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{name}: has a tangent, and there are no forward-mode derivatives")


def _rows(t, width, name, like=None):
    """[rows, width] of a tensor whose last dimension is the vector, in a layout that the kernels take."""
    if forward_ad._current_level >= 0:
        _no_tangent(t, name)
    shape = t.shape
    if not shape or shape[-1] != width:
        raise ValueError(f"{name}: the last dimension is {list(shape)[-1:]}, not {width}")
    if like is None:
        if t.dtype not in _TYPES:
            raise ValueError(f"{name}: {t.dtype} is not float32, bfloat16 or float16")
        if not t.is_cuda:
            raise ValueError(f"{name}: not on the GPU")
    elif t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name}: {t.dtype} on {t.device}, not {like.dtype} on {like.device}")
    if len(shape) == 2 and t.is_contiguous():
        return t
    if len(shape) != 2:
        t = t.reshape(-1, width)
    if (width > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < width):
        t = t.contiguous()
    return t


def _same_order(lead, like, name):
    """Leading dimensions of a tensor beside x's, `like`: the same, or rows in a line beside either."""
    if len(lead) > 1 and lead != like:
        a, b = [n for n in lead if n != 1], [n for n in like if n != 1]
        if a != b and len(a) > 1 and len(b) > 1:
            raise ValueError(f"{name}: leading dimensions {list(lead)}, not {list(like)}")


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _vector(t, n, name, dtype, device):
    if forward_ad._current_level >= 0:
        _no_tangent(t, name)
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name}: {list(t.shape)}, not [{n}]")
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name}: {t.dtype} on {t.device}, not {dtype} on {device}")
    return t.contiguous()


# ---- layer norm --------------------------------------------------------------------


def _norm_tensors(x, weight, bias):
    _need(x.dim() >= 1 and x.shape[-1] >= 1, "x: no last dimension")
    width = x.shape[-1]
    _sized(width, "x: the last dimension")
    x2 = _rows(x, width, "x")
    if weight.dtype != x.dtype and weight.dtype != torch.float32:
        raise ValueError(f"weight: {weight.dtype}, neither {x.dtype} nor float32")
    weight = _vector(weight, width, "weight", weight.dtype, x.device)
    if bias is not None:
        bias = _vector(bias, width, "bias", weight.dtype, x.device)
    return x2, weight, bias


def _norm_forward(x, weight, bias, eps, keep):
    x2, weight, bias = _norm_tensors(x, weight, bias)
    rows, width = x2.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = rstd = None
    if keep:
        mean = torch.empty(rows, dtype=torch.float32, device=x.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    _call("LayerNorm", LayerNormArgs(
        x=x2.data_ptr(), ldx=_ld(x2), weight=weight.data_ptr(), bias=None if bias is None else bias.data_ptr(),
        y=y.data_ptr(), ldy=width, mean=mean.data_ptr() if keep else None, rstd=rstd.data_ptr() if keep else None,
        rows=rows, width=width, type=_TYPES[x.dtype], paramType=_TYPES[weight.dtype], eps=eps), x.device)
    return y, mean, rstd


def layer_norm_forward(x, weight, bias=None, eps=1e-5):
    """(y, mean, rstd): the norm over the last dimension, and what its gradient needs of each row."""
    return _norm_forward(x, weight, bias, eps, True)


def layer_norm_backward(grad, x, weight, mean, rstd, has_bias=True):
    """(dx, dweight, dbias) of the norm; dbias is None without a bias."""
    x2, weight, _ = _norm_tensors(x, weight, None)
    rows, width = x2.shape
    _same_order(grad.shape[:-1], x.shape[:-1], "grad")
    g2 = _rows(grad, width, "grad", x)
    if g2.shape[0] != rows:
        raise ValueError(f"grad: {g2.shape[0]} rows, not {rows}")
    mean = _vector(mean, rows, "mean", torch.float32, x.device)
    rstd = _vector(rstd, rows, "rstd", torch.float32, x.device)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dweight = torch.empty_like(weight)
    dbias = torch.empty_like(weight) if has_bias else None
    _call("LayerNormGrad", LayerNormArgs(
        x=x2.data_ptr(), ldx=_ld(x2), weight=weight.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr(),
        dy=g2.data_ptr(), lddy=_ld(g2), dx=dx.data_ptr(), lddx=width,
        dweight=dweight.data_ptr(), dbias=dbias.data_ptr() if has_bias else None,
        rows=rows, width=width, type=_TYPES[x.dtype], paramType=_TYPES[weight.dtype]), x.device)
    return dx, dweight, dbias


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.has_bias = bias is not None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return layer_norm_backward(grad, *ctx.saved_tensors, has_bias=ctx.has_bias) + (None,)


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def layer_norm(x, weight, bias=None, eps=1e-5):
    """The norm of x over its last dimension."""
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _norm_forward(x, weight, bias, eps, False)[0]


# ---- gated feed-forward block ----------------------------------------------------------


_NO_COEF = (0.0, 0.0, 0.0, 0.0)


def _mlp_tensors(x, gate, up, down):
    _need(gate.dim() == 2 and up.dim() == 2 and down.dim() == 2, "gate, up and down are matrices")
    hidden, width = gate.shape
    _need(hidden >= 1 and width >= 1, "gate: no elements")
    _sized(hidden, "gate: rows")
    _sized(width, "gate: the last dimension")
    x2 = _rows(x, width, "x")
    gate, up, down = _rows(gate, width, "gate", x), _rows(up, width, "up", x), _rows(down, hidden, "down", x)
    if up.shape[0] != hidden:
        raise ValueError(f"up: {up.shape[0]} rows, not {hidden}")
    if down.shape[0] != width:
        raise ValueError(f"down: {down.shape[0]} rows, not {width}")
    return x2, gate, up, down


def _act(activation):
    """The number of an activation, and a cubic's coefficients."""
    if isinstance(activation, str):
        _need(activation in _ACTS, f"activation {activation!r}: neither silu, gelu nor four coefficients")
        return _ACTS[activation], _NO_COEF
    coef = tuple(float(c) for c in activation)
    _need(len(coef) == 4, "activation: a cubic has four coefficients, lowest degree first")
    return 2, coef


def _mlp_forward(x, gate, up, down, activation, keep):
    x2, gate, up, down = _mlp_tensors(x, gate, up, down)
    act, coef = _act(activation)
    rows, hidden, width = x2.shape[0], gate.shape[0], gate.shape[1]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    saved = g = u = None
    if keep:
        saved = torch.empty((2, rows, (hidden + 7) // 8 * 8), dtype=torch.float32, device=x.device)
        if rows:
            g = saved.data_ptr()
            u = g + 2 * saved.numel()
    _call("GatedMLP", GatedMLPArgs(
        x=x2.data_ptr(), ldx=_ld(x2), gate=gate.data_ptr(), ldgate=_ld(gate), up=up.data_ptr(), ldup=_ld(up), down=down.data_ptr(),
        lddown=_ld(down), y=y.data_ptr(), ldy=width, g=g, u=u, rows=rows, width=width, hidden=hidden, type=_TYPES[x.dtype], act=act,
        coef=coef), x.device)
    return y, saved


def gated_mlp_forward(x, gate, up, down, activation="silu"):
    """(y, saved): the block's output and, for its gradient, both projections in float32 (rounded
    to 16 bits they would cost the gradients more than their own rounding does)."""
    return _mlp_forward(x, gate, up, down, activation, True)


def gated_mlp_backward(grad, x, gate, up, down, saved, activation="silu"):
    """(dx, dgate, dup, ddown)."""
    x2, gate, up, down = _mlp_tensors(x, gate, up, down)
    act, coef = _act(activation)
    rows, hidden, width = x2.shape[0], gate.shape[0], gate.shape[1]
    _same_order(grad.shape[:-1], x.shape[:-1], "grad")
    g2 = _rows(grad, width, "grad", x)
    if g2.shape[0] != rows:
        raise ValueError(f"grad: {g2.shape[0]} rows, not {rows}")
    _need(tuple(saved.shape) == (2, rows, (hidden + 7) // 8 * 8) and saved.dtype == torch.float32 and saved.device == x.device
          and saved.is_contiguous(), "saved: not what the forward call returned")
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dgate, dup, ddown = (torch.empty(w.shape, dtype=x.dtype, device=x.device) for w in (gate, up, down))
    g = saved.data_ptr() if rows else None
    _call("GatedMLPGrad", GatedMLPArgs(
        x=x2.data_ptr(), ldx=_ld(x2), gate=gate.data_ptr(), ldgate=_ld(gate), up=up.data_ptr(), ldup=_ld(up), down=down.data_ptr(),
        lddown=_ld(down), g=g, u=g + 2 * saved.numel() if rows else None, dy=g2.data_ptr(), lddy=_ld(g2), dx=dx.data_ptr(), lddx=width,
        dgate=dgate.data_ptr(), dup=dup.data_ptr(), ddown=ddown.data_ptr(), rows=rows, width=width, hidden=hidden,
        type=_TYPES[x.dtype], act=act, coef=coef), x.device)
    return dx, dgate, dup, ddown


class _GatedMLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, up, down, activation):
        y, saved = gated_mlp_forward(x, gate, up, down, activation)
        ctx.save_for_backward(x, gate, up, down, saved)
        ctx.activation = activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return gated_mlp_backward(grad, *ctx.saved_tensors, ctx.activation) + (None,)


def gated_mlp(x, gate, up, down, activation="silu"):
    """The gated feed-forward block (act(x gate^T) * (x up^T)) down^T: gate, up [hidden, width], down [width, hidden].
    activation: "silu", "gelu" or a cubic's four coefficients, lowest degree first, which the block can also be
    evaluated with under encryption.  Hidden values and their gradients are factors of the next product, of x's type: in
    float16 one beyond 65504 is infinite, and gradients below 2^-14 lose bits unless the loss is scaled."""
    if _wants_grad(x, gate, up, down):
        return _GatedMLP.apply(x, gate, up, down, activation)
    return _mlp_forward(x, gate, up, down, activation, False)[0]


# ---- softmax cross entropy against a table ------------------------------------------------


def _loss_tensors(x, table, target, ignore_index):
    _need(table.dim() == 2 and table.shape[0] >= 1 and table.shape[1] >= 1, "table: not a matrix with elements")
    _sized(table.shape[0], "table: rows")
    _sized(table.shape[1], "table: the last dimension")
    _need(-(1 << 63) <= ignore_index < 1 << 63, "ignore_index: not an int64")
    _same_order(target.shape, x.shape[:-1], "target")
    x2 = _rows(x, table.shape[1], "x")
    target = _vector(target.reshape(-1) if target.dim() != 1 else target, x2.shape[0], "target", torch.int64, x.device)
    return x2, _rows(table, table.shape[1], "table", x), target


def cross_entropy_forward(x, table, target, ignore_index=-100):
    """(losses, lse), float32 for each row: the softmax cross entropy of x's products with the table's rows, and the
    logarithm of the softmax's sum.  Rows whose target is `ignore_index` have 0 for both; a target outside the table
    gives NaN.  The logits are never in memory."""
    x2, table, target = _loss_tensors(x, table, target, ignore_index)
    losses = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    lse = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _call("CrossEntropy", CrossEntropyArgs(
        x=x2.data_ptr(), ldx=_ld(x2), table=table.data_ptr(), ldtable=_ld(table), target=target.data_ptr(), loss=losses.data_ptr(),
        lse=lse.data_ptr(), rows=x2.shape[0], width=table.shape[1], vocab=table.shape[0], ignore=ignore_index,
        type=_TYPES[x.dtype]), x.device)
    return losses, lse


def cross_entropy_backward(grad, x, table, target, lse, ignore_index=-100):
    """(dx, dtable) for the gradient `grad` of the losses (float32); lse as the forward call gave it.  The logits are
    computed again, a piece of the table at a time."""
    x2, table, target = _loss_tensors(x, table, target, ignore_index)
    rows, width = x2.shape
    _same_order(grad.shape, x.shape[:-1], "grad")
    _same_order(lse.shape, x.shape[:-1], "lse")
    grad = _vector(grad.reshape(-1), rows, "grad", torch.float32, x.device)
    lse = _vector(lse.reshape(-1), rows, "lse", torch.float32, x.device)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dtable = torch.empty(table.shape, dtype=x.dtype, device=x.device)
    _call("CrossEntropyGrad", CrossEntropyArgs(
        x=x2.data_ptr(), ldx=_ld(x2), table=table.data_ptr(), ldtable=_ld(table), target=target.data_ptr(), lse=lse.data_ptr(),
        dloss=grad.data_ptr(), dx=dx.data_ptr(), lddx=width, dtable=dtable.data_ptr(), rows=rows, width=width, vocab=table.shape[0],
        ignore=ignore_index, type=_TYPES[x.dtype]), x.device)
    return dx, dtable


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, table, target, ignore_index):
        losses, lse = cross_entropy_forward(x, table, target, ignore_index)
        ctx.save_for_backward(x, table, target, lse)
        ctx.ignore_index = ignore_index
        return losses

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return cross_entropy_backward(grad, *ctx.saved_tensors, ctx.ignore_index) + (None, None)


def _total(losses, target, ignore_index):
    """(the losses' sum, or with a target their mean; what each one's gradient is of it).  (torch's sum of many values
    clears memory first, which a captured graph does not repeat.)"""
    total, factor = (torch.empty((), dtype=torch.float32, device=losses.device) for _ in "ab")
    if target is not None:
        target = target.reshape(-1).contiguous()
    _call("LossTotal", LossTotalArgs(
        loss=losses.data_ptr(), target=None if target is None else target.data_ptr(), total=total.data_ptr(), factor=factor.data_ptr(),
        rows=losses.numel(), ignore=ignore_index), losses.device)
    return total, factor


class _Total(torch.autograd.Function):
    @staticmethod
    def forward(ctx, losses, target, ignore_index):
        total, factor = _total(losses, target, ignore_index)
        ctx.save_for_backward(factor)
        ctx.shape = losses.shape
        return total

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return (grad * ctx.saved_tensors[0]).expand(ctx.shape), None, None


def cross_entropy(x, table, target, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of x [..., width] against table [vocab, width]: the mean over the rows that have a target
    (0 where none has one), their "sum", or "none" for a loss a row."""
    _need(reduction in ("mean", "sum", "none"), f"reduction {reduction!r}: neither mean, sum nor none")
    grad = _wants_grad(x, table)
    losses = _CrossEntropy.apply(x, table, target, ignore_index) if grad else cross_entropy_forward(x, table, target, ignore_index)[0]
    if reduction == "none":
        return losses
    target = target if reduction == "mean" else None
    return _Total.apply(losses, target, ignore_index) if grad else _total(losses, target, ignore_index)[0]
