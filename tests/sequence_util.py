"""The sequence operators in 64 bits on the CPU, from their definitions, and how far a kernel that
computes in fp32 may be from them.

Error bounds.  u = 2^-24 is the largest relative error of one fp32 rounding.  A bound is the same
formula run on magnitudes (every term replaced by its absolute value), times the roundings that a
value passes through; a scan's bound is a scan: if each row adds an error e[t], the state carries
E[t] = a[t] E[t-1] + e[t].  Values stored in the data's type get half a step of it on top,
finfo.eps / 2 relative to the value.
"""
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def wide(t):
    return None if t is None else t.detach().double().cpu()


def check(got, want, bound, dtype=None, what=""):
    """|got - want| <= bound + the rounding to ``dtype`` (of a value that is itself off by bound)."""
    got, want, bound = wide(got), want.detach(), bound.detach()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    dtype = dtype or torch.float32
    # below the smallest normal number a type's steps have one size
    limit = bound + half_step(dtype) * (want.abs() + bound) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    bad = ~((got - want).abs() <= limit)
    if bool(bad.any()):
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at {i}: got "
                             f"{got[i].item()!r}, want {want[i].item()!r}, limit {limit[i].item():.3g}")


def spans(B, T, offsets):
    """(batch index, first row, end row, state index) of every sequence."""
    if offsets is None:
        return [(b, 0, T, b) for b in range(B)]
    return [(0, offsets[j], offsets[j + 1], j) for j in range(len(offsets) - 1)]


# ---- recurrence --------------------------------------------------------------------------------

def recurrence(x, u, v, decay, scale, initial=None, offsets=None, dy=None, dfinal=None):
    """Outputs and bounds of the recurrence, as two dicts."""
    x, u, v, decay, initial, dy, dfinal = (wide(t) for t in (x, u, v, decay, initial, dy, dfinal))
    B, T, C = x.shape
    sp = torch.nn.functional.softplus(decay, threshold=60)
    r, i = torch.sigmoid(u), torch.sigmoid(v)
    z = scale * sp * r
    a = torch.exp(-z)
    beta = (-torch.expm1(-2 * z)).sqrt()
    b = beta * i * x
    n = len(offsets) - 1 if offsets is not None else B
    h0 = initial if initial is not None else torch.zeros(n, C, dtype=torch.float64)
    zero = torch.zeros(B, T, C, dtype=torch.float64)
    h, before, hbar, bbar, E = (zero.clone() for _ in range(5))
    state, sE = h0.clone(), torch.zeros(n, C, dtype=torch.float64)
    # Roundings per row.  b = beta i x: z (softplus to 2 units of 2^-23, its product with scale, r to
    # 3 units of 2^-23), 1 - e^-z (8), its root and two products: at most 32 u |b|.  a: |da| <= u (the
    # last rounding) + a z 16 u (through z) <= 7 u (z e^-z <= 0.37).  The state's own rounding: u.
    # P, the product of a's that carries a state over several rows, is off by no more than its a's
    # together.  Hence e = 32 u |b| + 9 u |h[t-1]|-magnitudes.
    for bi, s, e, j in spans(B, T, offsets):
        cur, mag, err = h0[j], h0[j].abs(), torch.zeros(C, dtype=torch.float64)
        for t in range(s, e):
            before[bi, t], bbar[bi, t] = cur, mag
            err = a[bi, t] * err + 32 * U * b[bi, t].abs() + 9 * U * mag
            cur = a[bi, t] * cur + b[bi, t]
            mag = a[bi, t] * mag + b[bi, t].abs()
            h[bi, t], hbar[bi, t], E[bi, t] = cur, mag, err + U * mag
        state[j], sE[j] = cur, err + U * mag
    out, tol = {"y": h, "state": state}, {"y": E, "state": sE}
    if dy is None:
        return out, tol
    q0 = dfinal if dfinal is not None else torch.zeros(n, C, dtype=torch.float64)
    g, gbar, Eg = (zero.clone() for _ in range(3))
    dinit, dinit_tol = q0.clone(), torch.zeros(n, C, dtype=torch.float64)
    for bi, s, e, j in spans(B, T, offsets):
        q, mag, err = q0[j], q0[j].abs(), torch.zeros(C, dtype=torch.float64)
        for t in reversed(range(s, e)):
            gt, gm = dy[bi, t] + q, dy[bi, t].abs() + mag
            g[bi, t], gbar[bi, t], Eg[bi, t] = gt, gm, err + 2 * U * gm
            err = a[bi, t] * (err + 2 * U * gm) + 9 * U * gm
            q, mag = a[bi, t] * gt, a[bi, t] * gm
        dinit[j], dinit_tol[j] = q, err
    inside = zero.clone()
    for bi, s, e, j in spans(B, T, offsets):
        inside[bi, s:e] = 1
    ix = i * x
    out["dx"] = g * beta * i
    tol["dx"] = beta * i * (Eg + 40 * U * gbar)
    out["dv"] = out["dx"] * x * (1 - i)
    # 1 - i: i to 3 units of 2^-23, absolutely
    tol["dv"] = x.abs() * ((1 - i) * tol["dx"] + 8 * U * gbar * beta * i)
    inner, inner_bar = a * a / beta * ix - a * before, a * a / beta * ix.abs() + a * bbar
    Eh = torch.zeros_like(E)
    for bi, s, e, j in spans(B, T, offsets):
        Eh[bi, s + 1:e] = E[bi, s:max(e - 1, s)]
    dz = g * inner
    # both terms carry a factor a = e^-z, whose relative error is z times z's own (16 u) and 4 u more; the
    # first term carries it twice
    dz_tol = (Eg + (48 + 32 * z) * U * gbar) * inner_bar + gbar * a * Eh
    dz_bar = gbar * inner_bar
    out["du"] = dz * z * (1 - r)
    tol["du"] = z * ((1 - r) * (dz_tol + 24 * U * dz_bar) + 8 * U * dz_bar)
    k = scale * torch.sigmoid(decay)
    # a sum of one fp32 per row: rows are added in groups, no value passes through more than 128 sums
    # at these lengths; sigmoid(decay) to 8 u
    out["ddecay"] = k * (dz * r * inside).sum((0, 1))
    tol["ddecay"] = k * ((dz_tol + (128 + 16) * U * dz_bar) * r * inside).sum((0, 1))
    out["dinitial"], tol["dinitial"] = dinit, dinit_tol
    for name in ("dx", "du", "dv"):
        out[name], tol[name] = out[name] * inside, tol[name] * inside
    return out, tol


# ---- convolution -------------------------------------------------------------------------------

ACTS = {
    None: lambda p: p,
    "relu": torch.relu,
    "relu6": lambda p: p.clamp(0, 6),
    "silu": lambda p: p * torch.sigmoid(p),
    "hardswish": lambda p: p * (p + 3).clamp(0, 6) / 6,
}


def conv(x, w, bias, act, initial=None, offsets=None, dy=None, dfinal=None):
    x, w, bias, initial, dy, dfinal = (wide(t) for t in (x, w, bias, initial, dy, dfinal))
    B, T, C = x.shape
    K = w.shape[2]
    n = len(offsets) - 1 if offsets is not None else B
    leaves = [x, w]
    h0 = initial if initial is not None else torch.zeros(n, K - 1, C, dtype=torch.float64)
    b0 = bias if bias is not None else torch.zeros(C, dtype=torch.float64)
    leaves += [b0, h0]
    for t in leaves:
        t.requires_grad_(dy is not None)

    def rows(x, w, b0, h0):
        """p, and the final rows, of every sequence."""
        p, final = x * 0, []
        for bi, s, e, j in spans(B, T, offsets):
            full = torch.cat([h0[j], x[bi, s:e]])
            if e > s:
                win = full.unfold(0, K, 1)                              # [rows, C, K]
                p = p.index_put((torch.tensor([bi]), torch.arange(s, e)), (win * w[:, 0]).sum(-1) + b0)
            final.append(full[full.shape[0] - (K - 1):])
        return p, torch.stack(final)

    inside = torch.zeros(B, T, 1, dtype=torch.float64)
    for bi, s, e, j in spans(B, T, offsets):
        inside[bi, s:e] = 1
    p, final = rows(x, w, b0, h0)
    y = ACTS[act](p) * inside
    pbar, _ = rows(x.detach().abs(), w.detach().abs(), b0.detach().abs(), h0.detach().abs())
    ptol = (K + 1) * U * pbar
    # activation: slope at most 1.1 (hard-swish 1.5); silu's sigmoid from an exponential that is off by
    # 2 + 1.16 |p| units of 2^-23, a sum and a quotient of 2 units
    sig = torch.sigmoid(p.detach())
    sig_tol = 2 * U * ((2 + 1.16 * p.detach().abs()) * sig * (1 - sig) + 4 * sig)
    slope = 1.5 if act == "hardswish" else 1.1
    ytol = slope * ptol + (p.detach().abs() * sig_tol if act == "silu" else 0) + 8 * U * y.detach().abs()
    out, tol = {"y": y, "state": final}, {"y": ytol * inside, "state": torch.zeros_like(final)}
    if dy is None:
        return {k: v.detach() for k, v in out.items()}, tol
    outs, given = [y], [dy]
    if dfinal is not None:
        outs.append(final)
        given.append(dfinal)
    grads = torch.autograd.grad(outs, leaves, given, allow_unused=True)
    grads = [torch.zeros_like(l) if g is None else g for g, l in zip(grads, leaves)]
    out.update(dx=grads[0], dweight=grads[1], dbias=grads[2], dinitial=grads[3])
    # dp = dy act'(p): the slope's own error through p (second derivative at most 0.5 for silu, 1/3 for
    # hard-swish) and its evaluation (8 roundings, and the sigmoid's)
    pd = p.detach()
    dptol = dy.abs() * (0.5 * ptol + 8 * U * 1.5 + (1 + pd.abs()) * 2 * sig_tol) * inside if act else 0 * pd
    dpbar = dy.abs() * 1.5 * inside if act else dy.abs() * inside
    wabs = w.detach().abs()
    with torch.enable_grad():
        # sums of magnitudes by the linear map's own adjoint
        xa, wa = x.detach().abs().requires_grad_(), wabs.clone().requires_grad_()
        ba, ha = b0.detach().abs().requires_grad_(), h0.detach().abs().requires_grad_()
        pa, fa = rows(xa, wa, ba, ha)
        fg = dfinal.abs() if dfinal is not None else torch.zeros_like(fa)
        # dw: 64 rows in a run, 8 runs, then the parts: no value passes through more than 128 sums here
        mags = torch.autograd.grad([pa, fa], [xa, wa, ba, ha], [dptol + 144 * U * dpbar, 2 * U * fg], allow_unused=True)
    mags = [torch.zeros_like(l) if g is None else g for g, l in zip(mags, leaves)]
    tol.update(dx=mags[0], dweight=mags[1], dbias=mags[2], dinitial=mags[3])
    return {k: v.detach() for k, v in out.items()}, tol


# ---- layer norm --------------------------------------------------------------------------------

def norm(x, w, b, eps, dy=None):
    x, w, b, dy = (wide(t) for t in (x, w, b, dy))
    C = x.shape[-1]
    w = torch.ones(C, dtype=torch.float64) if w is None else w
    b = torch.zeros(C, dtype=torch.float64) if b is None else b
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = (x - mean) * rstd
    # a row's sum: no value passes through more than 64 sums; x - mean inherits the mean's error, the
    # variance twice that relative to the deviation, the root 2 units
    mean_tol = 64 * U * x.abs().mean(-1, keepdim=True)
    rstd_rel = 64 * U + 2 * mean_tol * rstd
    xh_tol = rstd * (mean_tol + U * (x - mean).abs()) + xh.abs() * rstd_rel
    out = {"y": xh * w + b}
    tol = {"y": xh_tol * w.abs() + 2 * U * ((xh * w).abs() + b.abs())}
    if dy is None:
        return out, tol
    q = dy * w
    m1, m2 = q.mean(-1, keepdim=True), (q * xh).mean(-1, keepdim=True)
    inner = q - m1 - xh * m2
    out["dx"] = rstd * inner
    m1_tol = 66 * U * q.abs().mean(-1, keepdim=True)
    m2_tol = (q.abs() * xh_tol + 66 * U * (q * xh).abs()).mean(-1, keepdim=True)
    inner_tol = 4 * U * (q.abs() + m1.abs() + (xh * m2).abs()) + m1_tol + xh.abs() * m2_tol + xh_tol * m2.abs()
    tol["dx"] = rstd * inner_tol + out["dx"].abs() * rstd_rel
    rows = tuple(range(x.dim() - 1))
    out["dweight"], out["dbias"] = (dy * xh).sum(rows), dy.sum(rows)
    # rows in a CTA one after another, then the CTAs' parts: at most 128 sums at these sizes
    tol["dweight"] = (dy.abs() * xh_tol + 130 * U * (dy * xh).abs()).sum(rows)
    tol["dbias"] = 130 * U * dy.abs().sum(rows)
    return out, tol
