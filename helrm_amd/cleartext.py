"""Operators that train and score a model in the clear, on torch tensors.

The encrypted path (`orion_host`) evaluates a model that was trained: its
table, its Linears, its degree-3 activations.  These are the operators of
that training and of scoring beside it, on the same card:

    embedding       y[i] = scale * table[ids[i]]
    layer_norm      y = (x - mean) / sqrt(var + eps) * weight + bias
    gated_mlp       y = (act(x gate^T) * (x up^T)) down^T
    cross_entropy   log sum_v exp <x, table[v]> - <x, table[target]>
    distillation    the divergence of a teacher's top logits from the softmax of <x, table[v]>
    preference      log(1 + exp -m), m the difference of two sequences' log ratios to a reference

Each has a `_forward` and a `_backward` call, which a training loop of one's
own makes, and a form for torch's autograd.  The matrices' last dimension is
the vector; leading dimensions are rows.  Types: float32, bfloat16, float16,
one for all of an operator's tensors (a norm's weight and bias and a teacher's
logits may be float32 beside any; tokens' losses are float32); sums and softmax
statistics are float32.  Tensors of the same rows
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
import math

import torch
from torch.autograd import forward_ad

from .backend import (CrossEntropyArgs, DistillationArgs, EmbeddingArgs, GatedMLPArgs, HipError, LayerNormArgs, LossTotalArgs, PreferenceArgs,
                      load_library)

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
    for name in ("LayerNorm", "LayerNormGrad", "GatedMLP", "GatedMLPGrad", "CrossEntropy", "CrossEntropyGrad", "LossTotal",
                 "Distillation", "DistillationGrad", "Preference", "PreferenceGrad", "Embedding", "EmbeddingGrad"):
        call, size = getattr(lib, name), getattr(lib, name + "Workspace", None)
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
        if need:
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
    computed again, a piece of the table at a time.  Their gradient is a factor of two products: in 16-bit types of more than 64
    rows it is rounded to the type, and dx and dtable have that rounding and their own."""
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


# ---- distillation from a teacher's top logits ---------------------------------------------


def _teach_tensors(x, table, ids, temperature, ignore_index):
    _need(table.dim() == 2 and table.shape[0] >= 1 and table.shape[1] >= 1, "table: not a matrix with elements")
    _sized(table.shape[0], "table: rows")
    _sized(table.shape[1], "table: the last dimension")
    _need(-(1 << 63) <= ignore_index < 1 << 63, "ignore_index: not an int64")
    # (messages are made where they are needed: a shape's is a microsecond of a small call)
    if not 2.0 ** -60 <= temperature <= 2.0 ** 60:
        raise ValueError(f"temperature {temperature}: not positive, or out of range")
    if not (ids.dim() >= 1 and 1 <= ids.shape[-1] <= 1024):
        raise ValueError(f"ids: {list(ids.shape)}, not [..., top] with top from 1 to 1024")
    _same_order(ids.shape[:-1], x.shape[:-1], "ids")
    x2 = _rows(x, table.shape[1], "x")
    if ids.dtype != torch.int64 or ids.device != x.device:
        raise ValueError(f"ids: {ids.dtype} on {ids.device}, not {torch.int64} on {x.device}")
    ids = ids.reshape(-1, ids.shape[-1]).contiguous()
    if ids.shape[0] != x2.shape[0]:
        raise ValueError(f"ids: {ids.shape[0]} rows, not {x2.shape[0]}")
    return x2, _rows(table, table.shape[1], "table", x), ids


def distillation_forward(x, table, ids, logits, temperature=1.0, ignore_index=-100):
    """(losses, lse, saved), losses and lse float32 for each row: temperature^2 times the divergence of the teacher's softmax of
    logits / temperature over `ids` [..., top] from the softmax of x's products with all of the table's rows / temperature, and the
    logarithm of the latter's sum; saved is what the gradient needs.  An id that is `ignore_index` or has a logit of -inf is no
    entry, one that is there twice has both probabilities.  Rows without entries have 0 for both; an id outside the table gives
    NaN.  x's logits are never in memory."""
    x2, table, ids2 = _teach_tensors(x, table, ids, temperature, ignore_index)
    rows, top = ids2.shape
    if logits.shape != ids.shape:
        raise ValueError(f"logits: {list(logits.shape)}, not {list(ids.shape)}")
    if logits.dtype not in (x.dtype, torch.float32) or logits.device != x.device:
        raise ValueError(f"logits: {logits.dtype} on {logits.device}, neither {x.dtype} nor float32 on {x.device}")
    if forward_ad._current_level >= 0:
        _no_tangent(logits, "logits")
    logits = logits.reshape(rows, top).contiguous()
    losses = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    lse = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    kept = torch.empty(rows, dtype=torch.int64, device=x.device)
    held = torch.empty((3, rows, top), dtype=torch.float32, device=x.device)     # scores, probabilities, and int32 ids
    _call("Distillation", DistillationArgs(
        x=x2.data_ptr(), ldx=_ld(x2), table=table.data_ptr(), ldtable=_ld(table), ids=ids2.data_ptr(), logits=logits.data_ptr(),
        loss=losses.data_ptr(), lse=lse.data_ptr(), kept=kept.data_ptr(), scores=held.data_ptr(), probs=held.data_ptr() + 4 * rows * top,
        cols=held.data_ptr() + 8 * rows * top, rows=rows, width=table.shape[1], vocab=table.shape[0], top=top, type=_TYPES[x.dtype], teacherType=_TYPES[logits.dtype],
        ignore=ignore_index, temperature=temperature), x.device)
    return losses, lse, (kept, held)


def distillation_backward(grad, x, table, ids, lse, saved, temperature=1.0, ignore_index=-100):
    """(dx, dtable) for the gradient `grad` of the losses (float32); lse and saved as the forward call gave them.  The logits are
    computed again, a piece of the table at a time.  Their gradient is a factor of two products: in 16-bit types of more than 256
    rows it is rounded to the type, and dx and dtable have that rounding and their own."""
    x2, table, ids = _teach_tensors(x, table, ids, temperature, ignore_index)
    rows, width = x2.shape
    _same_order(grad.shape, x.shape[:-1], "grad")
    _same_order(lse.shape, x.shape[:-1], "lse")
    grad = _vector(grad.reshape(-1), rows, "grad", torch.float32, x.device)
    lse = _vector(lse.reshape(-1), rows, "lse", torch.float32, x.device)
    kept, held = saved
    _need(tuple(kept.shape) == (rows,) and kept.dtype == torch.int64 and kept.device == x.device and kept.is_contiguous()
          and tuple(held.shape) == (3, *ids.shape) and held.dtype == torch.float32 and held.device == x.device and held.is_contiguous(),
          "saved: not what the forward call returned")
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dtable = torch.empty(table.shape, dtype=x.dtype, device=x.device)
    _call("DistillationGrad", DistillationArgs(
        x=x2.data_ptr(), ldx=_ld(x2), table=table.data_ptr(), ldtable=_ld(table), lse=lse.data_ptr(), kept=kept.data_ptr(),
        scores=held.data_ptr(), probs=held.data_ptr() + 4 * ids.numel(), cols=held.data_ptr() + 8 * ids.numel(), dloss=grad.data_ptr(), dx=dx.data_ptr(), lddx=width,
        dtable=dtable.data_ptr(), rows=rows, width=width, vocab=table.shape[0], top=ids.shape[1], type=_TYPES[x.dtype],
        teacherType=_TYPES[x.dtype], ignore=ignore_index, temperature=temperature), x.device)
    return dx, dtable


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, table, ids, logits, temperature, ignore_index):
        losses, lse, (kept, held) = distillation_forward(x, table, ids, logits, temperature, ignore_index)
        ctx.save_for_backward(x, table, ids, lse, kept, held)
        ctx.rest = temperature, ignore_index
        ctx.mark_non_differentiable(kept)
        return losses, kept

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        x, table, ids, lse, kept, held = ctx.saved_tensors
        return distillation_backward(grad, x, table, ids, lse, (kept, held), *ctx.rest) + (None, None, None, None)


def distillation(x, table, ids, logits, temperature=1.0, ignore_index=-100, reduction="mean"):
    """Divergence of a teacher from x [..., width] against table [vocab, width], of the teacher's top logits [..., top] and their
    ids, both softmaxes at `temperature` and the loss times its square (distillation_forward has the formula): the mean over the
    rows that have a teacher (0 where none has one), their "sum", or "none" for a loss a row.  The teacher's logits have no
    gradient here."""
    _need(reduction in ("mean", "sum", "none"), f"reduction {reduction!r}: neither mean, sum nor none")
    _need(not _wants_grad(logits), "logits: require a gradient, and are the teacher's; detach them")
    grad = _wants_grad(x, table)
    if grad:
        losses, kept = _Distillation.apply(x, table, ids, logits, temperature, ignore_index)
    else:
        losses, _, (kept, _) = distillation_forward(x, table, ids, logits, temperature, ignore_index)
    if reduction == "none":
        return losses
    kept = kept if reduction == "mean" else None
    return _Total.apply(losses, kept, 0) if grad else _total(losses, kept, 0)[0]


# ---- pairs of sequences of which one is preferred ------------------------------------------


_KINDS = {"logistic": 0, "hinge": 1}


def _lines(t, like, name, dtype, packed):
    """(token values as the kernels take them, elements from one sequence's to the next's): of the shape and device of `like`."""
    if forward_ad._current_level >= 0:
        _no_tangent(t, name)
    if t.shape != like.shape:
        raise ValueError(f"{name}: {list(t.shape)}, not {list(like.shape)}")
    if t.dtype != dtype or t.device != like.device:
        raise ValueError(f"{name}: {t.dtype} on {t.device}, not {dtype} on {like.device}")
    length = t.shape[-1]
    if packed or t.is_contiguous():
        return t.contiguous(), length
    t = t.flatten(0, -2)
    if (length > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < length):
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else length


def _pairs(losses, target, offsets, ignore_index):
    """(leading dimensions of a pair, number of pairs, length, target and its ld, offsets)."""
    _need(-(1 << 63) <= ignore_index < 1 << 63, "ignore_index: not an int64")
    if losses.dtype != torch.float32:
        raise ValueError(f"losses: {losses.dtype}, not {torch.float32}")
    if offsets is None:
        if losses.dim() < 2 or losses.shape[-2] != 2:
            raise ValueError(f"losses: {list(losses.shape)}, not [..., 2, length]")
        lead = losses.shape[:-2]
        pairs = math.prod(lead)
    else:
        if losses.dim() != 1:
            raise ValueError(f"losses: {list(losses.shape)}, not [tokens] beside offsets")
        if offsets.dim() != 1 or offsets.shape[0] % 2 != 1:
            raise ValueError(f"offsets: {list(offsets.shape)}, not [2 * pairs + 1]")
        pairs = offsets.shape[0] // 2
        lead = (pairs,)
    if not losses.is_cuda:
        raise ValueError("losses: not on the GPU")
    if offsets is not None:
        offsets = _vector(offsets, 2 * pairs + 1, "offsets", torch.int64, losses.device)
    target, ld = (None, 0) if target is None else _lines(target, losses, "target", torch.int64, offsets is not None)
    return lead, pairs, losses.shape[-1], target, ld, offsets


def _values(t, name, device):
    if forward_ad._current_level >= 0:
        _no_tangent(t, name)
    if t.dtype != torch.float32 or t.device != device:
        raise ValueError(f"{name}: {t.dtype} on {t.device}, not {torch.float32} on {device}")
    return t.contiguous()


def _pointer(t):
    return None if t is None else t.data_ptr()


def _preference_forward(losses, reference, target, offsets, beta, margin, kind, smoothing, average, ignore_index, keep=True):
    if kind not in _KINDS:
        raise ValueError(f"kind {kind!r}: neither logistic nor hinge")
    _need(math.isfinite(beta) and math.isfinite(margin), "beta and margin are not finite")
    if not 0.0 <= smoothing <= (1.0 if kind == "logistic" else 0.0):
        raise ValueError(f"smoothing {smoothing}: not from 0 to 1, or not 0 with the hinge")
    lead, pairs, length, target, ldtarget, offsets = _pairs(losses, target, offsets, ignore_index)
    packed, device = offsets is not None, losses.device
    held, ldreference = (None, 0) if reference is None else _lines(reference, losses, "reference", torch.float32, packed)
    losses, ldloss = _lines(losses, losses, "losses", torch.float32, packed)
    values = torch.empty(lead, dtype=torch.float32, device=device)
    ratios = torch.empty((*lead, 2), dtype=torch.float32, device=device)
    slopes = torch.empty_like(ratios)
    kept = torch.empty(pairs, dtype=torch.int64, device=device) if keep else None
    _call("Preference", PreferenceArgs(
        loss=losses.data_ptr(), ldloss=ldloss, reference=_pointer(held), ldreference=ldreference, target=_pointer(target), ldtarget=ldtarget,
        offsets=_pointer(offsets), value=values.data_ptr(), ratio=ratios.data_ptr(), slope=slopes.data_ptr(), kept=_pointer(kept), pairs=pairs,
        length=length, ignore=ignore_index, kind=_KINDS[kind], average=bool(average), beta=beta, margin=margin, smoothing=smoothing), device)
    return values, ratios, slopes, kept


def preference_forward(losses, reference=None, target=None, offsets=None, beta=0.1, margin=0.0, kind="logistic", smoothing=0.0, average=False,
                       ignore_index=-100):
    """(values, ratios, slopes) of pairs of sequences whose first one is preferred: the pairs' losses [...], and for both sequences
    [..., 2] the sum of reference - losses over the tokens that count (their mean with `average`) and the derivative of the pair's
    value by each of those losses.  losses [..., 2, length] are the tokens' (float32, as cross_entropy gives them); or [tokens],
    sequence s the tokens from offsets[s] to offsets[s + 1].  Tokens whose target is `ignore_index` count in nothing.
    With m = beta * (ratio of the first - of the second) - margin: "logistic" (1 - smoothing) log(1 + exp -m) + smoothing log(1 +
    exp m), "hinge" max(0, 1 - m).  A pair without tokens that count has 0, one whose offsets descend or leave the tokens NaN."""
    return _preference_forward(losses, reference, target, offsets, beta, margin, kind, smoothing, average, ignore_index, False)[:3]


def preference_backward(grad, losses, slopes, target=None, offsets=None, ignore_index=-100):
    """The gradient of every token's loss, of losses' shape, for the gradient `grad` of the values; slopes as the forward call gave
    them.  Tokens that count in nothing have 0.  Of offsets that descend somewhere, a token has the gradient of one of the sequences
    that hold it, NaN or 0, the same on every run."""
    lead, pairs, length, target, ldtarget, offsets = _pairs(losses, target, offsets, ignore_index)
    device = losses.device
    if grad.shape != lead:
        raise ValueError(f"grad: {list(grad.shape)}, not {list(lead)}")
    if slopes.shape != (*lead, 2):
        raise ValueError(f"slopes: {list(slopes.shape)}, not {[*lead, 2]}")
    grad, slopes = (_values(t, name, device) for t, name in ((grad, "grad"), (slopes, "slopes")))
    d = torch.empty(losses.shape, dtype=torch.float32, device=device)
    _call("PreferenceGrad", PreferenceArgs(
        target=_pointer(target), ldtarget=ldtarget, offsets=_pointer(offsets), slope=slopes.data_ptr(), dvalue=grad.data_ptr(),
        dloss=d.data_ptr(), lddloss=length, pairs=pairs, length=length, ignore=ignore_index), device)
    return d


class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, losses, reference, target, offsets, ignore_index, rest):
        values, _, slopes, kept = _preference_forward(losses, reference, target, offsets, *rest, ignore_index)
        ctx.save_for_backward(losses, slopes, target, offsets)
        ctx.ignore_index = ignore_index
        ctx.mark_non_differentiable(kept)
        return values, kept

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        return (preference_backward(grad, *ctx.saved_tensors, ctx.ignore_index),) + (None,) * 5


def preference(losses, reference=None, target=None, offsets=None, beta=0.1, margin=0.0, kind="logistic", smoothing=0.0, average=False,
               ignore_index=-100, reduction="mean"):
    """Loss of pairs of sequences of which the first is preferred, from their tokens' losses and those of a reference model
    (preference_forward has the arguments and the formula): the mean over the pairs that have a token (0 where none has one), their
    "sum", or "none" for a loss a pair.  The reference has no gradient here."""
    _need(reduction in ("mean", "sum", "none"), f"reduction {reduction!r}: neither mean, sum nor none")
    _need(not _wants_grad(reference), "reference: requires a gradient, and is held; detach it")
    grad = _wants_grad(losses)
    rest = beta, margin, kind, smoothing, average
    if grad:
        values, kept = _Preference.apply(losses, reference, target, offsets, ignore_index, rest)
    else:
        values, _, _, kept = _preference_forward(losses, reference, target, offsets, *rest, ignore_index)
    if reduction == "none":
        return values
    kept = kept if reduction == "mean" else None
    return _Total.apply(values, kept, 0) if grad else _total(values, kept, 0)[0]


# ---- rows of a table for ids -----------------------------------------------------------------


def _embedding_ids(ids, vocab, ignore_index, device):
    _need(vocab >= 1, "table: no rows")
    _need(-(1 << 63) <= ignore_index < 1 << 63, "ignore_index: not an int64")
    if ids.dtype != torch.int64 or ids.device != device:
        raise ValueError(f"ids: {ids.dtype} on {ids.device}, not {torch.int64} on {device}")
    return ids.contiguous() if ids.dim() == 1 else ids.reshape(-1).contiguous()


def embedding_forward(ids, table, scale=1.0, ignore_index=-100):
    """table[ids] * scale, [..., width]: rows of zeros where an id is `ignore_index`, of NaN where another one is outside the table."""
    _need(table.dim() == 2 and table.shape[1] >= 1, "table: not a matrix with elements")
    vocab, width = table.shape
    _sized(vocab, "table: rows")
    _sized(width, "table: the last dimension")
    t2 = _rows(table, width, "table")
    flat = _embedding_ids(ids, vocab, ignore_index, table.device)
    y = torch.empty((*ids.shape, width), dtype=table.dtype, device=table.device)
    _call("Embedding", EmbeddingArgs(
        ids=flat.data_ptr(), table=t2.data_ptr(), ldtable=_ld(t2), y=y.data_ptr(), ldy=width, tokens=flat.shape[0], width=width,
        vocab=vocab, ignore=ignore_index, type=_TYPES[table.dtype], scale=scale), table.device)
    return y


def embedding_backward(grad, ids, vocab, scale=1.0, ignore_index=-100):
    """dtable [vocab, width] for the gradient `grad` [..., width] of the rows of `ids`, of grad's type: what ids outside the table
    and ignored ones have in grad goes nowhere."""
    _need(grad.dim() >= 1 and grad.shape[-1] >= 1, "grad: no last dimension")
    width = grad.shape[-1]
    _sized(width, "grad: the last dimension")
    _sized(vocab, "table: rows")
    _same_order(grad.shape[:-1], ids.shape, "grad")
    g2 = _rows(grad, width, "grad")
    flat = _embedding_ids(ids, vocab, ignore_index, grad.device)
    if flat.shape[0] != g2.shape[0]:
        raise ValueError(f"grad: {g2.shape[0]} rows, not {flat.shape[0]}")
    dtable = torch.empty((vocab, width), dtype=grad.dtype, device=grad.device)
    _call("EmbeddingGrad", EmbeddingArgs(
        ids=flat.data_ptr(), dy=g2.data_ptr(), lddy=_ld(g2), dtable=dtable.data_ptr(), tokens=flat.shape[0], width=width, vocab=vocab,
        ignore=ignore_index, type=_TYPES[grad.dtype], scale=scale), grad.device)
    return dtable


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, ignore_index):
        ctx.save_for_backward(ids)
        ctx.rest = table.shape[0], scale, ignore_index
        return embedding_forward(ids, table, scale, ignore_index)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return None, embedding_backward(grad, *ctx.saved_tensors, *ctx.rest), None, None


def embedding(ids, table, scale=1.0, ignore_index=-100):
    """Rows of table [vocab, width] for ids of any shape, times `scale`: [..., width].  The table's gradient is the sum of its ids'
    rows in float32, rounded once, and the same on every run."""
    if _wants_grad(table):
        return _Embedding.apply(ids, table, scale, ignore_index)
    return embedding_forward(ids, table, scale, ignore_index)
