"""Plain 64-bit implementations of the cleartext operators on the CPU, each
result with a bound on the error that an implementation of the stated
precision may have: `(value, size)`, size the same sum with every term's
absolute value.  A sum of K float32 terms is within (K + 1) 2^-24 of its
size, a value rounded to a type of unit roundoff u within u of it."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
CUBIC = (-0.0320, 0.2195, 0.5706, 0.2048)   # lowest degree first


def d(t):
    return t.detach().cpu().double()


def act(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        p = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    c = name
    return c[0] + g * (c[1] + g * (c[2] + g * c[3])), c[1] + g * (2 * c[2] + g * 3 * c[3])


def layer_norm(x, w, b, eps):
    x, w = d(x), d(w)
    mu = x.mean(1, keepdim=True)
    r = ((x - mu).square().mean(1, keepdim=True) + eps).rsqrt()
    h = (x - mu) * r
    return h * w + (0 if b is None else d(b)), mu[:, 0], r[:, 0], h


def layer_norm_grad(dy, x, w, eps):
    _, _, r, h = layer_norm(x, w, None, eps)
    dy, w = d(dy), d(w)
    t = dy * w
    dx = r[:, None] * (t - t.mean(1, keepdim=True) - h * (t * h).mean(1, keepdim=True))
    return dx, (dy * h).sum(0), dy.sum(0)


def mlp(x, gate, up, down, name):
    x, gate, up, down = d(x), d(gate), d(up), d(down)
    g, u = x @ gate.T, x @ up.T
    a, _ = act(name, g)
    return (a * u) @ down.T


def mlp_grad(dy, x, gate, up, down, name):
    dy, x, gate, up, down = d(dy), d(x), d(gate), d(up), d(down)
    g, u = x @ gate.T, x @ up.T
    a, da = act(name, g)
    dh = dy @ down
    dg, du = dh * u * da, dh * a
    return dg @ gate + du @ up, dg.T @ x, du.T @ x, dy.T @ (a * u)


def mlp_sizes(dy, x, gate, up, down, name):
    """Sizes of y, dx, dgate, dup, ddown: every product and sum with absolute values."""
    dy, x, gate, up, down = (d(t).abs() for t in (dy, x, gate, up, down))
    g, u = x @ gate.T, x @ up.T
    # |act(g)| <= |g|, |act'| <= 1.2 for silu and gelu
    if isinstance(name, str):
        a, da = g, torch.full_like(g, 1.2)
    else:
        c = [abs(v) for v in name]
        a, da = c[0] + g * (c[1] + g * (c[2] + g * c[3])), c[1] + g * (2 * c[2] + g * 3 * c[3])
    dh = dy @ down
    dg, du = dh * u * da, dh * a
    return (a * u) @ down.T, dg @ gate + du @ up, dg.T @ x, du.T @ x, dy.T @ (a * u)


def cross_entropy(x, table, target, ignore=-100):
    """(losses, lse)."""
    x, table, target = d(x), d(table), target.cpu()
    losses, lse = torch.zeros(len(x), dtype=torch.float64), torch.zeros(len(x), dtype=torch.float64)
    for t in range(len(x)):
        k = int(target[t])
        if k == ignore:
            continue
        z = table @ x[t]
        lse[t] = torch.logsumexp(z, 0)
        losses[t] = lse[t] - z[k] if 0 <= k < len(table) else math.nan
    return losses, lse


def cross_entropy_grad(grad, x, table, target, ignore=-100):
    """(dx, dtable, both with absolute values in every sum, and both with the softmax itself in the place of the
    logits' gradient: an error e of a logit changes softmax - onehot by softmax * e, however small the difference)."""
    x, table, target, grad = d(x), d(table), target.cpu(), d(grad)
    rows = torch.nonzero(target != ignore)[:, 0]
    p = torch.softmax(x[rows] @ table.T, 1)
    soft = p * grad[rows, None].abs()
    p[torch.arange(len(rows)), target[rows]] -= 1
    p *= grad[rows, None]
    dx, sx, px = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    dx[rows], sx[rows], px[rows] = p @ table, p.abs() @ table.abs(), soft @ table.abs()
    return dx, p.T @ x[rows], sx, p.abs().T @ x[rows].abs(), px, soft.T @ x[rows].abs()


def check(got, want, size, tol, what):
    """|got - want| <= tol * size everywhere, NaN where want is NaN."""
    got, want = d(got), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in the wrong places"
    off = torch.nan_to_num((got - want).abs() - tol * size, nan=0.0)
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 0, f"{what}: {((got - want).abs() / (tol * size + 1e-300)).nan_to_num(0).max().item():.2f} times the bound"
