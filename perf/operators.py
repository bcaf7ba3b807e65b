"""The block operators' cases: what is timed, in plain torch operations and through ``ffn_ops``.

Three operators: the RMS norm with the residual's addition (16-bit or e4m3 output, and its backward
pass), the gated linear recurrence along packed sequences (and its backward pass), and the matrix
products of rows grouped by expert (forward, both gradients, and the e4m3 forward).
"""
import math
import sys
from pathlib import Path

import torch

own = False

PKG = Path(__file__).resolve().parents[1] / "ffnerf-experimental_b200"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
E4M3_MAX = 448.0
EPS = 1e-6


def _ops():
    if str(PKG) not in sys.path:
        sys.path.insert(0, str(PKG))
    import ffn_ops
    return ffn_ops


# --------------------------------------------------------------------------------------- the cases
def _norm(n, d, type, out="same", group=0, residual=True, train=False):
    return {"op": "norm", "n": n, "d": d, "type": type, "out": out, "group": group, "residual": residual,
            "train": train}


def _scan(seqs, steps, d, type, form="sigmoid", ragged=False, initial=False, reverse=False, train=False):
    return {"op": "scan", "seqs": seqs, "steps": steps, "d": d, "type": type, "form": form, "ragged": ragged,
            "initial": initial, "reverse": reverse, "train": train}


def _experts(n, experts, k, m, type, train=False, skew=1.0):
    return {"op": "experts", "n": n, "experts": experts, "k": k, "m": m, "type": type, "train": train, "skew": skew}


def listed():
    return [
        # one sample's feature row: the latency of a single call
        {"name": "norm: one row", **_norm(1, 1024, "bf16")},
        # rendering a wide trunk: rows quantised for the experts' 8-bit product, one scale a row
        {"name": "norm: 8 bits per row", **_norm(16384, 4096, "bf16", out="e4m3")},
        # samples at the framework's own hidden width, a scale for each 32 columns, no residual stream
        {"name": "norm: width 64, 8 bits", **_norm(262144, 64, "fp16", out="e4m3", group=32, residual=False)},
        # a training step's rows at an odd count and a width that is no multiple of a vector of lanes
        {"name": "norm: train, odd", **_norm(49999, 1000, "bf16", train=True)},
        # samples that arrive one at a time, the state carried by the caller
        {"name": "scan: one step", **_scan(256, 1, 1024, "bf16", initial=True)},
        # back-to-front compositing of 64-wide features over 64 samples a ray, 2^20 samples
        {"name": "scan: rays, train", **_scan(16384, 64, 64, "fp16", reverse=True, train=True)},
        # few very long sequences: the length has to be split
        {"name": "scan: long, train", **_scan(2, 32768, 1024, "bf16", train=True)},
        # rays with their own number of samples, some with none, in full precision
        {"name": "scan: ragged", **_scan(1500, 1000, 200, "fp32", form="linear", ragged=True, initial=True)},
        # a few rows over the experts: the weights' bytes count
        {"name": "experts: 16 rows", **_experts(16, 8, 2048, 2048, "bf16")},
        # a training step of wide experts
        {"name": "experts: train", **_experts(16384, 16, 1024, 4096, "bf16", train=True)},
        # 8-bit rows against 8-bit weights, an odd number of rows
        {"name": "experts: 8 bits", **_experts(30011, 8, 4096, 2048, "e4m3")},
        # the framework's hidden width and step size: 2^20 samples, 64 regions
        {"name": "experts: width 64, train", **_experts(1 << 20, 64, 64, 64, "fp16", train=True)},
    ]


def _log(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return v + 1 if v == 3072 else v


def _log8(rng, lo, hi, step=8):
    v = max(1, _log(rng, lo, hi) // step) * step
    return v + step if v == 3072 else v


def draw(rng):
    op = rng.choice(("norm", "scan", "experts"))
    if op == "norm":
        out = rng.choice(("same", "e4m3"))
        group = rng.choice((0, 32, 64, 128)) if out == "e4m3" else 0
        d = _log8(rng, max(64, group), 8192, group or 1)
        return _norm(_log(rng, 1, (1 << 25) // d), d, rng.choice(("bf16", "fp16", "fp32")), out, group,
                     rng.random() < 0.7, out == "same" and rng.random() < 0.5)
    if op == "scan":
        d = _log(rng, 16, 2048)
        steps = _log(rng, 1, min(32768, (1 << 25) // d))
        return _scan(_log(rng, 1, max(1, (1 << 25) // (d * steps))), steps, d, rng.choice(("bf16", "fp16", "fp32")),
                     rng.choice(("sigmoid", "linear")), rng.random() < 0.3, rng.random() < 0.5, rng.random() < 0.3,
                     rng.random() < 0.5)
    type = rng.choice(("bf16", "fp16", "e4m3"))
    step = 1 if type != "e4m3" and rng.random() < 0.25 else 16   # any width, or what 8-bit rows need
    k, m = _log8(rng, 64, 4096, step), _log8(rng, 64, 4096, step)
    experts = _log(rng, 1, 64)
    while experts * k * m > 1 << 28:
        experts = max(1, experts // 2)
    n = _log(rng, 1, min(1 << 20, (1 << 36) // (k * m), (1 << 30) // (k + m)))
    return _experts(n, experts, k, m, type, type != "e4m3" and rng.random() < 0.5, rng.choice((1.0, 2.0)))


# -------------------------------------------------------------------------------------- the inputs
def _counts(case, seed):
    """Rows of each expert: shares u^skew of uniform draws u, so skew 2 leaves some experts almost bare."""
    g = torch.Generator().manual_seed(seed * 7 + 3)
    share = torch.rand(case["experts"], generator=g, dtype=torch.float64).add_(0.25).pow(2 * case["skew"])
    ends = (share.cumsum(0) / share.sum() * case["n"]).round().long()
    ends[-1] = case["n"]
    return [0] + ends.tolist()


def _lengths(case, seed):
    if not case["ragged"]:
        return [case["steps"]] * case["seqs"]
    # the same lengths for every seed, in an order of its own: 0 to `steps`, none for rays that miss the scene
    g = torch.Generator().manual_seed(case["steps"])
    n = torch.randint(0, case["steps"] + 1, (case["seqs"],), generator=g)
    n[torch.rand(case["seqs"], generator=g) < 0.05] = 0
    n[0] = case["steps"]
    return n[torch.randperm(case["seqs"], generator=g.manual_seed(seed * 5 + 1))].tolist()


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    s = {"case": case}
    if case["op"] == "norm":
        n, d, t = case["n"], case["d"], TYPES[case["type"]]
        s["x"] = rand(n, d).mul_(rand(n, 1).exp_()).to(t)      # rows of very different size
        s["residual"] = rand(n, d).to(t) if case["residual"] else None
        s["gamma"] = 1 + 0.2 * rand(d)
        if case["train"]:
            s["dy"] = rand(n, d).to(t)
            s["dresidual"] = rand(n, d).to(t) if case["residual"] else None
    elif case["op"] == "scan":
        t, d, lens = TYPES[case["type"]], case["d"], _lengths(case, seed)
        n = sum(lens)
        s["offsets"] = torch.tensor([0] + lens).cumsum(0).to("cuda", torch.int32)
        gate = rand(n, d).mul_(1.5).add_(2.0)                   # sigmoid gates about 0.88
        s["gate"] = (gate if case["form"] == "sigmoid" else gate.sigmoid_()).to(t)
        s["value"] = rand(n, d).to(t)
        s["h0"] = rand(case["seqs"], d) if case["initial"] else None
        if case["train"]:
            s["dh"] = rand(n, d).to(t)
            s["dh_last"] = rand(case["seqs"], d)
    else:
        n, e, k, m = case["n"], case["experts"], case["k"], case["m"]
        s["offsets"] = torch.tensor(_counts(case, seed)).to("cuda", torch.int32)
        s["cap"] = max(b - a for a, b in zip(_counts(case, seed), _counts(case, seed)[1:]))
        x, w = rand(n, k), rand(e, m, k).mul_(k ** -0.5)
        if case["type"] == "e4m3":
            s["x_scale"] = x.abs().amax(1).clamp_min_(1e-20).div_(E4M3_MAX)
            s["w_scale"] = w.abs().amax(2).div_(E4M3_MAX)
            s["x"] = x.div_(s["x_scale"][:, None]).to(torch.float8_e4m3fn)
            s["w"] = w.div_(s["w_scale"][:, :, None]).to(torch.float8_e4m3fn)
        else:
            s["x"], s["w"] = x.to(TYPES[case["type"]]), w.to(TYPES[case["type"]])
            if case["train"]:
                s["dy"] = rand(n, m).to(TYPES[case["type"]])
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ---------------------------------------------------------------------- through the framework's calls
def _run_own(s):
    c, ops = s["case"], _ops()
    if c["op"] == "norm":
        if c["out"] == "e4m3":
            y, h, _, scale = ops.rmsnorm(s["x"], s["gamma"], s["residual"], eps=EPS, out="e4m3", group=c["group"])
            return {"y": y, "scale": scale, "h": h if c["residual"] else None}
        y, h, rstd, _ = ops.rmsnorm(s["x"], s["gamma"], s["residual"], eps=EPS)
        r = {"y": y, "h": h if c["residual"] else None}
        if c["train"]:
            r["dx"], r["dgamma"] = ops.rmsnorm_bwd(s["dy"], h, s["gamma"], rstd, s["dresidual"])
        return r
    if c["op"] == "scan":
        # packed sequences with their offsets, or [sequence, step, channel] where all are alike
        lay = (lambda v: v) if c["ragged"] else (lambda v: v.view(c["seqs"], c["steps"], c["d"]))  # noqa: E731
        kw = {"form": c["form"], "reverse": c["reverse"], "h0": s["h0"]}
        if c["ragged"]:
            kw.update(offsets=s["offsets"], max_len=c["steps"])
        gate, value = lay(s["gate"]), lay(s["value"])
        h, last = ops.gated_scan(gate, value, **kw)
        r = {"h": h.view(-1, c["d"]), "last": last}
        if c["train"]:
            dgate, dvalue, dh0 = ops.gated_scan_bwd(lay(s["dh"]), gate, value, h, dh_last=s["dh_last"], **kw)
            r["dgate"], r["dvalue"] = dgate.view(-1, c["d"]), dvalue.view(-1, c["d"])
            if c["initial"]:
                r["dh0"] = dh0
        return r
    if c["type"] == "e4m3":
        return {"y": ops.expert_mm(s["x"], s["w"], s["offsets"], x_scale=s["x_scale"], w_scale=s["w_scale"])}
    r = {"y": ops.expert_mm(s["x"], s["w"], s["offsets"])}
    if c["train"]:
        r["dx"], r["dw"] = ops.expert_mm_bwd(s["dy"], s["x"], s["w"], s["offsets"])
    return r


# ---------------------------------------------------------------------------------- the plain forms
def _quantise(y, group):
    n, d = y.shape
    z = y.view(n, d // (group or d), group or d)
    scale = z.abs().amax(-1) / E4M3_MAX
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    q = (z / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(n, d)
    return q, (scale if group else scale[:, 0])


def _plain_norm(s):
    c, t = s["case"], s["x"].dtype
    h = s["x"].float()
    if c["residual"]:
        h = h + s["residual"].float()
    rstd = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    xhat = h * rstd
    y = xhat * s["gamma"]
    if c["out"] == "e4m3":
        q, scale = _quantise(y, c["group"])
        return {"y": q, "scale": scale, "h": h.to(t) if c["residual"] else None}
    r = {"y": y.to(t), "h": h.to(t) if c["residual"] else None}
    if c["train"]:
        dy = s["dy"].float()
        u = dy * s["gamma"]
        dx = rstd * (u - xhat * (u * xhat).mean(1, keepdim=True))
        if c["residual"]:
            dx = dx + s["dresidual"].float()
        r["dx"], r["dgamma"] = dx.to(t), (dy * xhat).sum(0)
    return r


def _prefix(a, b, most):
    """All of b_t + a_t b_{t-1} + a_t a_{t-1} b_{t-2} + ... by doubling; a is zero where a sequence begins."""
    step = 1
    while step < most:   # log2 of the longest sequence: each turn doubles the steps that an entry spans
        b = torch.cat((b[:step], b[step:] + a[step:] * b[:-step]))
        a = torch.cat((a[:step], a[step:] * a[:-step]))
        step *= 2
    return b


def _plain_scan(s):
    c, t, off = s["case"], s["gate"].dtype, s["offsets"].long()
    turn = (lambda v: v.flip(0)) if c["reverse"] else (lambda v: v)  # noqa: E731
    n, seqs = s["gate"].shape[0], c["seqs"]
    begin, end = off[:-1], off[1:]
    if c["reverse"]:
        begin, end = (n - end).flip(0), (n - begin).flip(0)
    full = end > begin
    first, final = begin[full], end[full] - 1
    gate, value = turn(s["gate"]).float(), turn(s["value"]).float()
    a = gate.sigmoid() if c["form"] == "sigmoid" else gate
    b = value * (1 - a) if c["form"] == "sigmoid" else value
    h0 = torch.zeros(seqs, c["d"], device=a.device) if s["h0"] is None else turn(s["h0"])
    inner = a.index_fill(0, first, 0.0)
    h = _prefix(inner, b.index_add(0, first, a[first] * h0[full]), c["steps"])
    last = h0.clone()
    last[full] = h[final]
    r = {"h": turn(h).to(t), "last": turn(last)}
    if c["train"]:
        before = torch.cat((h[:1], h[:-1])).index_copy(0, first, h0[full])
        dlast = turn(s["dh_last"])
        top = turn(s["dh"]).float().index_add(0, final, dlast[full])
        after = torch.cat((inner[1:], inner[:1])).index_fill(0, final, 0.0)
        grad = _prefix(after.flip(0), top.flip(0), c["steps"]).flip(0)
        if c["form"] == "sigmoid":
            r["dgate"] = turn(grad * (before - value) * a * (1 - a)).to(t)
            r["dvalue"] = turn(grad * (1 - a)).to(t)
        else:
            r["dgate"], r["dvalue"] = turn(grad * before).to(t), turn(grad).to(t)
        if c["initial"]:
            dh0 = dlast.clone()
            dh0[full] = a[first] * grad[first]
            r["dh0"] = turn(dh0)
    return r


def _plain_experts(s):
    c, off = s["case"], s["offsets"].long()
    e, cap, n = c["experts"], s["cap"], c["n"]
    row = torch.arange(n, device=off.device)
    expert = torch.searchsorted(off[1:], row, right=True)
    slot = expert * cap + row - off[expert]
    spread = lambda v: v.new_zeros(e * cap, v.shape[1]).index_copy(0, slot, v).view(e, cap, -1)  # noqa: E731
    gather = lambda v: v.view(e * cap, -1)[slot]  # noqa: E731
    x, w = s["x"].float(), s["w"].float()
    if c["type"] == "e4m3":
        x, w = x * s["x_scale"][:, None], w * s["w_scale"][:, :, None]
        return {"y": gather(spread(x) @ w.transpose(1, 2)).to(torch.bfloat16)}
    t = s["x"].dtype
    xs = spread(x)
    r = {"y": gather(xs @ w.transpose(1, 2)).to(t)}
    if c["train"]:
        dys = spread(s["dy"].float())
        r["dx"], r["dw"] = gather(dys @ w).to(t), (dys.transpose(1, 2) @ xs).to(t)
    return r


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _plain_norm, "scan": _plain_scan, "experts": _plain_experts}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------ work and truth
def work(case):
    if case["op"] == "norm":
        n, d, z = case["n"], case["d"], SIZE[case["type"]]
        e = n * d
        out = e * (1 if case["out"] == "e4m3" else z) + (4 * n * (d // (case["group"] or d)) if case["out"] == "e4m3" else 0)
        b = e * z * (3 if case["residual"] else 1) + out + 4 * d
        f = 6 * e
        if case["train"]:
            # h is read back in the backward pass: a user's backward pass comes later than its forward pass
            b += e * z * (4 if case["residual"] else 3) + 8 * d + 8 * n
            f += 10 * e
        return {"bytes": b, "flops": f}
    if case["op"] == "scan":
        n = sum(_lengths(case, 0))
        e, z, q = n * case["d"], SIZE[case["type"]], 4 * case["seqs"] * case["d"]
        b, f = 3 * e * z + q * (2 if case["initial"] else 1), 6 * e
        if case["train"]:
            b += e * z * (6 if case["form"] == "sigmoid" else 5) + q * (3 if case["initial"] else 1)
            f += 12 * e
        return {"bytes": b, "flops": f}
    n, e, k, m = case["n"], case["experts"], case["k"], case["m"]
    z = 1 if case["type"] == "e4m3" else 2
    live = min(e, n)                                       # experts that have rows
    b = n * k * z + live * k * m * z + n * m * 2
    f = 2 * n * k * m
    if case["train"]:
        b += 2 * n * (2 * m + 2 * k) + 2 * k * m * (live + e)
        f *= 3
    return {"bytes": b, "flops": f}


def _exact_norm(c, s):
    h = s["x"].double() + (s["residual"].double() if c["residual"] else 0)
    g, d = s["gamma"].double(), c["d"]
    norm = h.square().sum(1).div(d).add(EPS).sqrt()
    y = torch.einsum("nd,d,n->nd", h, g, 1 / norm)
    keep = h if c["residual"] else None
    if c["out"] == "e4m3":
        w = c["group"] or d
        scale = torch.stack([y[:, i:i + w].abs().max(1).values for i in range(0, d, w)], 1) / E4M3_MAX
        scale[scale == 0] = 1
        return {"y": None, "scale": scale if c["group"] else scale[:, 0], "h": keep}
    r = {"y": y, "h": keep}
    if c["train"]:
        dy = s["dy"].double()
        # y_j = g_j h_j / norm and d norm / d h_i = h_i / (d norm)
        dot = torch.einsum("nd,d,nd->n", dy, g, h)
        dx = dy * g / norm[:, None] - h * (dot / (d * norm ** 3))[:, None]
        r["dx"] = dx + s["dresidual"].double() if c["residual"] else dx
        r["dgamma"] = torch.einsum("nd,nd,n->d", dy, h, 1 / norm)
    return r


def _exact_scan(c, s):
    lens = torch.tensor(_lengths(c, s["seed"]))
    most, seqs, d, dev = int(lens.max()), c["seqs"], c["d"], "cuda"
    if most > 40000 or seqs * most * d > 1 << 29:
        return None
    off = [0] + lens.cumsum(0).tolist()
    # one step of every sequence at a time, in the order in which it goes; place[t] are the rows of step t
    live = [torch.nonzero(lens > t)[:, 0] for t in range(most)] if c["ragged"] else [torch.arange(seqs)] * most
    start = torch.tensor(off[:-1])
    place = [(start[i] + (lens[i] - 1 - t if c["reverse"] else t)) for t, i in enumerate(live)]
    if not c["ragged"]:
        i = torch.arange(seqs, device=dev)
        live, sd = [i] * most, start.to(dev)
        place = [sd + (most - 1 - t if c["reverse"] else t) for t in range(most)]
    else:
        live, place = [i.to(dev) for i in live], [p.to(dev) for p in place]
    sig = c["form"] == "sigmoid"

    def at(p):
        g, v = s["gate"][p].double(), s["value"][p].double()
        a = 1 / (1 + (-g).exp()) if sig else g
        return a, v, (1 / (1 + g.exp()) if sig else None)

    state = torch.zeros(seqs, d, dtype=torch.float64, device=dev) if s["h0"] is None else s["h0"].double()
    init = state.clone()
    h = torch.zeros(off[-1], d, dtype=torch.float64, device=dev)
    for i, p in zip(live, place):
        a, v, na = at(p)
        state[i] = a * state[i] + (na * v if sig else v)
        h[p] = state[i]
    r = {"h": h, "last": state}
    if c["train"]:
        carry = s["dh_last"].double()
        dg, dv = torch.zeros_like(h), torch.zeros_like(h)
        for t in range(most - 1, -1, -1):
            i, p = live[t], place[t]
            a, v, na = at(p)
            before = h[p + (1 if c["reverse"] else -1)] if t else init[i]
            gr = carry[i] + s["dh"][p].double()
            dg[p] = gr * (before - v) * a * na if sig else gr * before
            dv[p] = gr * na if sig else gr
            carry[i] = a * gr
        r["dgate"], r["dvalue"] = dg, dv
        if c["initial"]:
            r["dh0"] = carry
    return r


def _exact_experts(c, s):
    ends = _counts(c, s["seed"])
    y = torch.zeros(c["n"], c["m"], dtype=torch.float64, device="cuda")
    r = {"y": y}
    if c["train"]:
        r["dx"] = torch.zeros(c["n"], c["k"], dtype=torch.float64, device="cuda")
        r["dw"] = torch.zeros(c["experts"], c["m"], c["k"], dtype=torch.float64, device="cuda")
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        if b == a:
            continue
        x, w = s["x"][a:b].double(), s["w"][e].double()
        if c["type"] == "e4m3":
            x, w = x * s["x_scale"][a:b, None].double(), w * s["w_scale"][e][:, None].double()
        torch.mm(x, w.t(), out=y[a:b])
        if c["train"]:
            dy = s["dy"][a:b].double()
            torch.mm(dy, w, out=r["dx"][a:b])
            torch.mm(dy.t(), x, out=r["dw"][e])
    return r


def exact(case, seed):
    s = _inputs(case, seed)
    s["seed"] = seed
    return {"norm": _exact_norm, "scan": _exact_scan, "experts": _exact_experts}[case["op"]](case, s)
