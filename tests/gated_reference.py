"""The gated scan in float64 by its definition, token by token, with a bound on what 32-bit arithmetic may be off.

A float32 evaluation of h = a h' + b in any grouping is off by at most K * 2^-24 * M, where M sums, over all tokens that reach an
element, the absolute values that pass through each rounding: M[t] = |a| M[t-1] + |a| H[t-1] + |b|, H[t] = |a| H[t-1] + |b|.  K counts the
roundings per token in units of 2^-24: the gate's factors (fp32: exp 4, sum 1, quotient 1, difference 1; 16-bit inputs, where the exponential is
the fast one, 2 + 1.16 |gate| ulp = 22 units at |gate| = 8 and the quotient 4), the product with u 1, the fma 1, and as many again for the product of factors
that carries a state over a run of rows.
"""
import torch

UNIT = 2.0 ** -24
K = {torch.float32: 16.0, torch.float16: 64.0, torch.bfloat16: 64.0}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def factors(gate, form):
    if form == "sigmoid":
        return torch.sigmoid(gate), torch.sigmoid(-gate)
    if form == "log":
        return torch.exp(gate), -torch.expm1(gate)
    return gate, 1 - gate


def scan(u, gate, h0, form, weighted):
    """(length, dim) -> y, h_last, by a loop over the tokens (differentiable)."""
    a, c = factors(gate, form)
    b = c * u if weighted else u
    h, ys = h0, []
    for t in range(u.shape[0]):
        h = a[t] * h + b[t]
        ys.append(h)
    return (torch.stack(ys) if ys else u.clone()), h


def _bound(a, b, h0, reverse=False):
    """H and M of the recurrence above."""
    H, M = h0.abs(), torch.zeros_like(h0)
    hs, ms = [], []
    order = range(a.shape[0] - 1, -1, -1) if reverse else range(a.shape[0])
    for t in order:
        M = a[t] * M + a[t] * H + b[t]
        H = a[t] * H + b[t]
        hs.append(H)
        ms.append(M)
    if reverse:
        hs.reverse(), ms.reverse()
    return torch.stack(hs), torch.stack(ms)


def expected(u, gate, h0, dy, dlast, form, weighted, dtype):
    """One sequence: {name: (value, tolerance)} of y, h_last, du, dgate, dh0 (float64, (length, dim) or (dim,))."""
    zero = torch.zeros(u.shape[1], dtype=torch.float64)
    u, gate, dy = (t.detach().double().cpu() for t in (u, gate, dy))
    h0 = zero if h0 is None else h0.detach().double().cpu()
    dlast = zero if dlast is None else dlast.detach().double().cpu()
    if u.shape[0] == 0:
        e = torch.zeros_like(u)
        return {"y": (e, e), "h_last": (h0, zero), "du": (e, e), "dgate": (e, e), "dh0": (dlast, zero)}
    lu, lg, lh = (t.clone().requires_grad_(True) for t in (u, gate, h0))
    y, last = scan(lu, lg, lh, form, weighted)
    du, dgate, dh0 = torch.autograd.grad([y, last], [lu, lg, lh], [dy, dlast])
    y, last = y.detach(), last.detach()
    a, c = factors(gate, form)
    b = (c * u if weighted else u).abs()
    a, c = a.abs(), c.abs()
    H, M = _bound(a, b, h0)
    Hp, Mp = torch.cat([h0.abs()[None], H[:-1]]), torch.cat([zero[None], M[:-1]])
    # dh[t] = dy[t] + a[t+1] dh[t+1]
    an = torch.cat([a[1:], torch.ones_like(a[:1])])
    G, N = _bound(an, dy.abs(), dlast, reverse=True)
    slope = {"sigmoid": a * c, "log": a, "direct": torch.ones_like(a)}[form]
    w = c if weighted else torch.ones_like(c)
    inner = Hp + u.abs() if weighted else Hp
    k, r = K[dtype] * UNIT, half_step(dtype)
    tol = {"y": k * M, "h_last": k * M[-1], "du": k * (N + 2 * G) * w,
           "dgate": k * slope * ((N + 3 * G) * inner + G * Mp), "dh0": k * a[0] * (N[0] + 2 * G[0])}
    val = {"y": y, "h_last": last, "du": du, "dgate": dgate, "dh0": dh0}
    # a value below the type's normal range is off by half of its smallest step
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return {n: (val[n], tol[n] * (1 + r) + (r * val[n].abs() + tiny if n in ("y", "du", "dgate") and dtype != torch.float32 else 1e-38)) for n in val}


def check(name, got, want):
    value, tol = want
    err = (got.detach().double().cpu() - value).abs()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert torch.isfinite(err).all(), name
    over = err > tol
    assert not over.any(), f"{name}: {int(over.sum())} of {err.numel()} off, worst {float((err / tol.clamp_min(1e-300)).max()):.3g} of the bound"
