"""The block operators in 64 bits, step by step, with bounds on what fp32 arithmetic may be off by."""
import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half an ulp, relative
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}   # half a subnormal step


def norm(x, gamma, residual, eps):
    h = x.double() + (residual.double() if residual is not None else 0)
    rstd = 1 / (h.square().mean(1) + eps).sqrt()
    return h, rstd, h * rstd[:, None] * gamma.double()


def norm_rel(d):
    """Relative error of an fp32 row factor: a thread adds at most d / 64 + 32 squares in a row, then a
    tree of ten; the root halves it; the three products and rsqrt add five units."""
    return 2.0 ** -24 * (d / 64 + 32 + 10 + 5)


def norm_bwd(dy, h, gamma, rstd, dresidual):
    dy, h, s = dy.double(), h.double(), rstd.double()[:, None]
    xhat, u = h * s, dy * gamma.double()
    mean = (u * xhat).mean(1, keepdim=True)
    dx = s * (u - xhat * mean)
    size = s * (u.abs() + xhat.abs() * (u * xhat).abs().mean(1, keepdim=True))
    if dresidual is not None:
        dx, size = dx + dresidual.double(), size + dresidual.double().abs()
    return dx, size, (dy * xhat).sum(0), (dy * xhat).abs().sum(0)


def _gate(g, form):
    if form == "linear":
        return g, torch.ones_like(g)
    return torch.sigmoid(g), torch.sigmoid(-g)


def scan(gate, value, h0, offsets, form, reverse):
    """h, h_last and the bound of the fp32 state's error (units of its own rounding, delta per step)."""
    n, d = gate.shape
    a, na = _gate(gate.double(), form)
    b = value.double() * na
    delta = 2.0 ** -20 if form == "sigmoid" else 2.0 ** -22     # exp: two ulp and |g| 2^-24 1.44; products
    h, err = torch.zeros(n, d, dtype=torch.float64), torch.zeros(n, d, dtype=torch.float64)
    last = torch.zeros(len(offsets) - 1, d, dtype=torch.float64)
    lerr = torch.zeros_like(last)
    for s in range(len(offsets) - 1):
        x = h0[s].double().clone() if h0 is not None else torch.zeros(d, dtype=torch.float64)
        e = torch.zeros(d, dtype=torch.float64)
        rows = range(offsets[s], offsets[s + 1])
        for r in (reversed(rows) if reverse else rows):
            e = a[r].abs() * e + delta * ((a[r] * x).abs() + b[r].abs())
            x = a[r] * x + b[r]
            h[r], err[r] = x, e
        last[s], lerr[s] = x, e
    return h, last, 4 * err, 4 * lerr


def scan_bwd(dh, dh_last, gate, value, h, h0, offsets, form, reverse):
    n, d = gate.shape
    a, na = _gate(gate.double(), form)
    delta = 2.0 ** -20 if form == "sigmoid" else 2.0 ** -22
    v, hh = value.double(), h.double()
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)  # noqa: E731
    dg, dv, eg, ev = z(n, d), z(n, d), z(n, d), z(n, d)
    dh0, e0 = z(len(offsets) - 1, d), z(len(offsets) - 1, d)
    for s in range(len(offsets) - 1):
        m = dh_last[s].double().clone() if dh_last is not None else z(d)
        e = z(d)
        rows = list(range(offsets[s], offsets[s + 1]))
        if reverse:
            rows.reverse()
        for i in range(len(rows) - 1, -1, -1):
            r = rows[i]
            before = hh[rows[i - 1]] if i else (h0[s].double() if h0 is not None else z(d))
            size = dh[r].double().abs() + m.abs()
            g, e = dh[r].double() + m, e + delta * size
            if form == "sigmoid":
                dg[r], dv[r] = g * (before - v[r]) * a[r] * na[r], g * na[r]
                eg[r] = (e * (before - v[r]).abs() + 2 * delta * size * (before.abs() + v[r].abs())) * a[r] * na[r]
                ev[r] = (e + delta * size) * na[r]
            else:
                dg[r], dv[r], eg[r], ev[r] = g * before, g, (e + delta * size) * before.abs(), e
            m, e = a[r] * g, a[r].abs() * (e + delta * size)
        dh0[s], e0[s] = m, e
    return dg, dv, dh0, 4 * eg, 4 * ev, 4 * e0


def experts(x, w, offsets):
    """y and, per result, the sum of its terms' magnitudes."""
    n, m = x.shape[0], w.shape[1]
    y, size = (torch.zeros(n, m, dtype=torch.float64, device=x.device) for _ in range(2))
    for e in range(w.shape[0]):
        a, b = offsets[e], offsets[e + 1]
        if b > a:
            xe, we = x[a:b].double(), w[e].double()
            y[a:b], size[a:b] = xe @ we.t(), xe.abs() @ we.abs().t()
    return y, size


def within(got, want, bound, dtype):
    """Every element within `bound` of `want`, plus one rounding to `dtype`."""
    got, want, bound = got.double().cpu(), want.cpu(), bound.cpu()
    tol = bound * (1 + UNIT[dtype]) + UNIT[dtype] * want.abs() + TINY[dtype]
    off = (got - want).abs()
    assert torch.isfinite(got).all()
    worst = float((off - tol).max()) if off.numel() else 0.0
    assert worst <= 0, f"over its bound by {worst:.3g}; largest difference {float(off.max()):.3g}"
