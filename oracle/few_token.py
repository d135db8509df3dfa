"""CPU / 64-bit restatement of the few-token operators (4-bit weights, mixtures of experts), with error bounds.
TEST INFRASTRUCTURE ONLY (tests/): never imported by the package.

Every function returns (value, bound) in float64: the value of the definition and how far a right kernel may be off it.
The bounds count, term by term,
  * the rounding of the output, and of the hidden state between the two kernels, to the 16-bit type:
    eps / 2 of the value, plus half the smallest subnormal;
  * 32-bit sums: each addition is off by at most 2^-23 of the sum of magnitudes S = sum |w| |x| so far (the tensor
    core may truncate, hence 2^-23 and not 2^-24); a sum of n columns in groups of G takes at most n / 16 steps of the
    matrix instruction (16 columns each, counted as 2 additions) and n / G of the group sums, and at most 32 joins;
  * 4-bit products only: an activation enters as a sum of three e5m2 numbers that is off by at most 2^-31 of the largest
    activation of its token and group (up to 4 tokens), or of its token (a token's rows of all experts in the down
    projection of a mixture);
  * the gate activation in 32 bits: 2^-19 relative (exp and division of the fast kind, each below 2^-21), and
    its slope, at most 1.13 for every activation here.
"""
from __future__ import annotations

import torch
from torch import Tensor

SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)
TERM_FLOOR = 2.0 ** -31


def unpack(w4: Tensor, scale: Tensor, zero: Tensor | None) -> Tensor:
    """float64 [.., rows, cols] of the packed format, nibble by nibble from the bytes."""
    b = w4.to(torch.int64).unflatten(-1, (-1, 4))
    word = b[..., 0] + (b[..., 1] << 8) + (b[..., 2] << 16) + (b[..., 3] << 24)
    q = torch.stack([(word >> s) & 15 for s in SHIFTS], dim=-1).flatten(-2).double()
    group = q.shape[-1] // scale.shape[-2]
    s = scale.double().repeat_interleave(group, dim=-2).transpose(-1, -2)
    z = 8.0 if zero is None else (zero & 15).double().repeat_interleave(group, dim=-2).transpose(-1, -2)
    return (q - z) * s


def _half_step(v: Tensor, dt: torch.dtype) -> Tensor:
    f = torch.finfo(dt)
    return v.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def _block_largest(x: Tensor, group: int) -> Tensor:
    """The value that the error of an element's terms is relative to."""
    if x.shape[0] <= 4:
        return _largest(x, group)
    return x.abs().amax(-1, keepdim=True).expand_as(x)


def _largest(x: Tensor, group: int) -> Tensor:
    """|x| of every element replaced by the largest of its group of columns."""
    return x.abs().unflatten(-1, (-1, group)).amax(-1, keepdim=True).expand(*x.shape[:-1], -1, group).flatten(-2)


def product(x: Tensor, w: Tensor, group: int = 0, largest: Tensor | None = None):
    """x w^T in 64 bits and the bound of its 32-bit sums (group > 0: on 4-bit weights with that group size). A 4-bit
    product adds up q and takes the zero point off at the end: its magnitudes are up to (15 + 15) scale, where the
    group's largest |w| is at least 7.5 scale (weights made by a quantiser that uses the range): 4 times that."""
    v = x @ w.transpose(-1, -2)
    n = w.shape[-1]
    steps = n / 8 + (n / group if group else 0) + 32
    if not group:
        return v, (x.abs() @ w.abs().transpose(-1, -2)) * (steps * 2.0 ** -23)
    size = 4 * _largest(w, group)
    return v, (x.abs() @ size.transpose(-1, -2)) * (steps * 2.0 ** -23) + \
        ((_block_largest(x, group) if largest is None else largest) @ size.transpose(-1, -2)) * TERM_FLOOR


_ACTS = {
    "silu": torch.nn.functional.silu, "swish": torch.nn.functional.silu, "no_act": lambda v: v, "relu": torch.relu,
    "gelu": torch.nn.functional.gelu, "sigmoid": torch.sigmoid, "tanh": torch.tanh,
    "leaky_relu": lambda v: torch.nn.functional.leaky_relu(v, 0.01),
}


def hidden(x: Tensor, wg: Tensor, bg, wu: Tensor, bu, act: str, group: int = 0, largest: Tensor | None = None):
    """act(x wg^T + bg) * (x wu^T + bu) before its rounding, and the bound."""
    g, dg = product(x, wg, group, largest)
    u, du = product(x, wu, group, largest)
    g = g if bg is None else g + bg
    u = u if bu is None else u + bu
    a = _ACTS[act](g)
    da = 1.13 * dg + a.abs() * 2.0 ** -19 + 2.0 ** -23 * g.abs()
    return a * u, da * u.abs() + a.abs() * du + da * du + (a * u).abs() * 2.0 ** -22


def finish(y: Tensor, dy: Tensor, bias, residual, dt: torch.dtype):
    for t in (bias, residual):
        if t is not None:
            y = y + t
            dy = dy + (y.abs() + t.abs()) * 2.0 ** -23
    return y, dy + _half_step(y, dt)


def linear(x, w, bias, residual, dt, group: int = 0):
    y, dy = product(x.double(), w, group)
    d = lambda t: None if t is None else t.double()
    return finish(y, dy, d(bias), d(residual), dt)


def mlp(x, wg, bg, wu, bu, wd, bd, residual, dt, act="silu", group: int = 0):
    d = lambda t: None if t is None else t.double()
    h, dh = hidden(x.double(), wg, d(bg), wu, d(bu), act, group)
    dh = dh + _half_step(h, dt)
    y, dy = product(h, wd, group)
    return finish(y, dy + dh @ wd.abs().t(), d(bd), d(residual), dt)


def route(x, w_router, top_k: int, renormalize: bool):
    """(ids, weights) from 64-bit logits; equal logits: lower index first."""
    logits = x.double() @ w_router.double().t()
    p = torch.softmax(logits, -1)
    ids = torch.sort(logits, dim=-1, descending=True, stable=True)[1][:, :top_k]
    w = torch.gather(p, 1, ids)
    return ids.to(torch.int32), (w / w.sum(1, keepdim=True) if renormalize else w)


def moe(x, ids, weights, wg, wu, wd, residual, dt, act="silu", group: int = 0):
    """Experts' weights in float64 ([experts, rows, cols]); ids outside the range skipped."""
    x = x.double()
    E, T = wg.shape[0], x.shape[0]
    valid = (ids >= 0) & (ids < E)
    share = torch.zeros((T, E), dtype=torch.float64, device=x.device)
    share.scatter_add_(1, ids.long().clamp(0, E - 1), torch.where(valid, weights.double(), torch.zeros_like(weights).double()))
    hit = torch.zeros((T, E), dtype=torch.bool, device=x.device)
    for j in range(ids.shape[1]):
        rows = torch.nonzero(valid[:, j])[:, 0]
        hit[rows, ids[rows, j].long()] = True
    top = torch.where(valid, weights.double().abs(), torch.zeros_like(weights).double()).amax(1, keepdim=True)
    y, dy = torch.zeros_like(x), torch.zeros_like(x)
    active = int(hit.any(0).sum())
    x_largest = _block_largest(x, group) if group else None
    parts = []
    for e in range(E):
        t = torch.nonzero(hit[:, e])[:, 0]
        if len(t) == 0:
            continue
        h, dh = hidden(x[t], wg[e], None, wu[e], None, act, group, None if x_largest is None else x_largest[t])
        f = torch.where(top[t] > 0, share[t, e][:, None] / top[t], torch.zeros_like(top[t]))
        h, dh = h * f, dh * f.abs() + (h * f).abs() * 2.0 ** -22
        parts.append((e, t, h, dh + _half_step(h, dt)))
    # what a token's hidden values are relative to when they become terms: their group, or all its hidden values
    token_largest = torch.zeros((T, 1), dtype=torch.float64, device=x.device)
    for e, t, h, dh in parts:
        token_largest[t] = torch.maximum(token_largest[t], h.abs().amax(1, keepdim=True))
    for e, t, h, dh in parts:
        largest = None
        if group:
            largest = _largest(h, group) if T <= 4 else token_largest[t].expand_as(h)
        y[t] += top[t] * (h @ wd[e].t())
        # one sum over all active experts: its steps count for every part
        own = product(h, wd[e], group, largest)[1]
        dy[t] += top[t] * (dh @ wd[e].abs().t() + own * active)
    return finish(y, dy + y.abs() * 2.0 ** -22, None, None if residual is None else residual.double(), dt)


def check(got: Tensor, want: Tensor, bound: Tensor, what: str) -> None:
    got, want, bound = got.double().cpu(), want.cpu(), bound.cpu()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} != {tuple(want.shape)}"
    off = (got - want).abs() / bound
    worst = float(torch.nan_to_num(off, nan=float("inf")).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound at {int(off.argmax())} ({float(got.flatten()[off.argmax()])} " \
                         f"for {float(want.flatten()[off.argmax()])})"


# ------------------------------------------------------------------------------- root-mean-square error of 4-bit products --
# The bounds above are worst cases and grow with the square of the columns: over thousands of columns they hide a product
# of the wrong precision. These limits are for the root-mean-square error over a token's outputs and grow like the root.
#
# The output's own rounding is taken out of the way by a residual: with residual = -round(y) the kernel returns
# y - round(y), whose rounding is off by eps / 2 of at most eps / 2 of y.
def as_terms(x: Tensor, group: int, terms: int = 3, largest: Tensor | None = None) -> Tensor:
    """The float64 values that stand for x in a 4-bit product: per block (see _block_largest; `largest` where it is wider)
    a power of two brings the largest magnitude to [2^14, 2^15), and each term is the e5m2 rounding of what is left. CPU."""
    block = _block_largest(x, group) if largest is None else largest.expand_as(x)
    e = 14 - torch.frexp(block)[1] + 1
    up = torch.ldexp(torch.ones_like(x), torch.where(block > 0, e, torch.zeros_like(e)).clamp_max(120))
    rest, total = x * up, torch.zeros_like(x)
    for _ in range(terms):
        t = rest.float().to(torch.float8_e5m2).double()
        rest, total = rest - t, total + t
    return total / up


def rms(v: Tensor) -> Tensor:
    """Of every token's (row's) values."""
    return v.double().pow(2).mean(-1).sqrt()


def product_rms_limit(x: Tensor, scale: Tensor, y: Tensor, extra: float = 0.0) -> Tensor:
    """Largest root-mean-square error over a token's outputs y = x w^T (float64 x [M, cols], scale [groups, rows]).

    A group's sum is made by up to 12 steps of the matrix instruction (128 columns, 32 a step, three terms), each off by at
    most 2^-23 of the sum so far, all perhaps to the same side (a tensor core that truncates); the integers q are at most
    15, and over inputs without a pattern the sum of q x is at most 15 |x_g| in the mean, |x_g| the length of the
    group's activations. sx is a sum of up to 13 rounded steps (eight columns, five exchanges) times at most 15, and two
    roundings apply it: 12 + 13 / 2 + 1 < 20 such steps, 300 * 2^-23 of scale |x_g|. Errors of different groups have nothing
    to do with each other and add up like a root, and so do the roundings of the sums over groups: at most cols / group
    + 34 of them, half of 2^-23 of y each. The terms are off by TERM_FLOOR of the largest activation, times 15 scale."""
    groups, cols = scale.shape[-2], x.shape[-1]
    s2 = scale.double().pow(2)
    lengths = x.unflatten(-1, (groups, -1)).pow(2).sum(-1)
    inner = 300 * 2.0 ** -23 * (lengths @ s2).mean(-1).sqrt()
    floor = TERM_FLOOR * 15 * x.abs().amax(-1) * (s2.sum(0).mean() * (cols // groups)).sqrt()
    return inner + floor + rms(y) * (2.0 ** -24 * (groups + 34) ** 0.5 + extra)


def hidden_rounded(x: Tensor, wg: Tensor, sg: Tensor, bg, wu: Tensor, su: Tensor, bu, act: str, dt: torch.dtype,
                   f: Tensor | None = None):
    """The hidden state of a 4-bit MLP as the kernel rounds it between its halves (times f), and the variance of what the
    errors d before that rounding make of it: a value changes its rounding with a probability of at most d / step, by a
    step (and by d where that is larger): d (step + d). d: the products' root-mean-square limits through the activation
    (slope at most 1.13), and 2^-18 of the value for the activation itself and the products around it."""
    g, u = x @ wg.t(), x @ wu.t()
    dg, du = product_rms_limit(x, sg, g)[:, None], product_rms_limit(x, su, u)[:, None]
    g = g if bg is None else g + bg.double()
    u = u if bu is None else u + bu.double()
    a = _ACTS[act](g)
    h = a * u
    d = 1.13 * dg * u.abs() + a.abs() * du + h.abs() * 2.0 ** -18
    if f is not None:
        h, d = h * f, d * f.abs()
    info = torch.finfo(dt)
    return h.to(dt).double(), d * (h.abs() * info.eps + info.smallest_normal * info.eps + d)


def mlp_rms(x, wg, sg, bg, wu, su, bu, wd, sd, bd, dt, act="silu"):
    """(y, limit) of decode_fwd_w4 without a residual: weights in float64, scales as they are stored."""
    h, var = hidden_rounded(x.double(), wg, sg, bg, wu, su, bu, act, dt)
    y = h @ wd.t()
    limit = product_rms_limit(h, sd, y) + (var @ wd.pow(2).t()).mean(-1).sqrt()
    return (y if bd is None else y + bd.double()), limit + (0 if bd is None else rms(bd[None]) * 2.0 ** -23)


def moe_rms(x, ids, weights, wg, sg, wu, su, wd, sd, dt, act="silu"):
    """(y, limit) of moe_decode_fwd_w4 without a residual, every id valid and once in its token."""
    x, weights, T, E = x.double(), weights.double(), x.shape[0], wg.shape[0]
    top = weights.abs().amax(1, keepdim=True)
    parts, largest = [], torch.zeros((T, 1), dtype=torch.float64, device=x.device)
    for e in range(E):
        t, place = torch.nonzero(ids == e, as_tuple=True)
        if len(t):
            h, var = hidden_rounded(x[t], wg[e], sg[e], None, wu[e], su[e], None, act, dt, weights[t, place][:, None] / top[t])
            largest[t] = torch.maximum(largest[t], h.abs().amax(1, keepdim=True))
            parts.append((e, t, h, var))
    y, square = torch.zeros_like(x), torch.zeros(T, dtype=torch.float64, device=x.device)
    for e, t, h, var in parts:   # errors of different experts add up like a root; the floor is that of the token's largest
        part = h @ wd[e].t()
        y[t] += top[t] * part
        widest = TERM_FLOOR * 15 * largest[t, 0] * (sd[e].double().pow(2).sum(0).mean() * (h.shape[1] // sd.shape[-2])).sqrt()
        own = product_rms_limit(h, sd[e], part) + widest
        square[t] += top[t, 0].pow(2) * (own.pow(2) + (var @ wd[e].pow(2).t()).mean(-1))
    groups = len(parts) * sd.shape[-2]
    return y, square.sqrt() + rms(y) * 2.0 ** -24 * (groups + 34) ** 0.5


def cancelling_residual(y: Tensor, dt: torch.dtype) -> Tensor:
    return (-y).to(dt)


def check_rms(got: Tensor, y: Tensor, residual: Tensor, limit: Tensor, dt: torch.dtype, what: str,
              rows: Tensor | None = None) -> None:
    """`got` = y + residual in `dt`, residual = cancelling_residual(y): root-mean-square error of every token (over the
    outputs `rows`) against its limit and the rounding of what is left of y, eps / 2 of eps / 2 of it."""
    left = y + residual.double()
    err, y = got.double() - left, y if rows is None else y[:, rows]
    off = rms(err if rows is None else err[:, rows]) / (limit + rms(y) * (torch.finfo(dt).eps ** 2 / 4))
    worst = float(torch.nan_to_num(off, nan=float("inf")).max())
    assert worst <= 1.0, f"{what}: root-mean-square error {worst:.3g} times its limit at token {int(off.argmax())}"
