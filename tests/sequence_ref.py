"""fp64 references of the sequence operators with the error each output may have.

Every reference returns {output: (value, bound)}.  The bounds count roundings, they are
not fitted: U = 2^-24 is half a step of fp32, and an output that is stored in a 16-bit type
adds torch.finfo(type).eps / 2 of its own magnitude.

Scans.  One step contributes a relative error of at most EPS to each of its two terms:
a rounding of the product A, one of the sum, each at most three times over (thread, warp
and tile folds) = 6 U, and for the gates G: __expf is off by 2 + 1.173 |x| ulp (12 ulp for
|x| <= 8), the sum and the reciprocal of the sigmoid 2 more, so sigmoid and the exponent L
by 14 ulp, sqrt(1 - a^2) by half of twice that plus 4 for its series and root, b by the sum
of sqrt, sigmoid and two products: under 36 ulp = 72 U; a itself by |L| * 14 ulp + 14 ulp.
An error made at one step is carried on by the later steps' factors like the state
itself, so the error of h_t is at most EPS * W_t with W_t = |a_t| (W_{t-1} + |h|_{t-1}) + |b_t|,
|h|_t = |a_t| |h|_{t-1} + |b_t|.
"""
import torch

U = 2.0 ** -24
GATE = 72 * U


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _walk(a, b, h0):
    """h_t = a_t h_{t-1} + b_t over dim 0; returns (all h_t, all h_{t-1})."""
    hs, prev, h = [], [], h0
    for t in range(a.shape[0]):
        prev.append(h)
        h = a[t] * h + b[t]
        hs.append(h)
    return torch.stack(hs), torch.stack(prev)


def _one_sequence(op, args, h0, dh, dlast, scale):
    """Time-first fp64 tensors of one batch of equally long sequences."""
    if op == "linear":
        a, b = args["a"], args["b"]
        eps = 6 * U
    else:
        x, s, q = args["x"], torch.sigmoid(args["rate"]), torch.sigmoid(args["gate"])
        L = -scale * torch.nn.functional.softplus(args["decay"], threshold=1000.0) * s
        a = L.exp()
        beta = (-torch.expm1(2 * L)).sqrt()
        b = beta * q * x
        eps = 6 * U + GATE * (1 + L.abs().max().item())
    h, prev = _walk(a, b, h0)
    mag, mag_prev = _walk(a.abs(), b.abs(), h0.abs())
    W, W_prev = _walk(a.abs(), a.abs() * mag_prev + b.abs(), torch.zeros_like(h0))
    out = {"h": (h, eps * W), "state": (h[-1], eps * W[-1])}
    if dh is None:
        return out

    def back(g, last):  # c_t = a_t lambda_t, lambda_t = g_t + c_{t+1}
        lam, c = [None] * a.shape[0], last
        for t in range(a.shape[0] - 1, -1, -1):
            lam[t] = g[t] + c
            c = a[t] * lam[t]
        return torch.stack(lam), c

    lam, dh0 = back(dh, dlast)
    aa = a.abs()
    m, WL, c, cw = [None] * len(aa), [None] * len(aa), dlast.abs(), torch.zeros_like(dlast)
    for t in range(len(aa) - 1, -1, -1):
        m[t], WL[t] = dh[t].abs() + c, cw + dh[t].abs() + c
        c, cw = aa[t] * m[t], aa[t] * (WL[t] + m[t])
    m, WL = torch.stack(m), torch.stack(WL)
    out["dh0"] = (dh0, eps * cw)
    if op == "linear":
        out["da"] = (lam * prev, eps * (WL * mag_prev + m * (W_prev + mag_prev)))
        out["db"] = (lam, eps * WL)
        return out
    # products of at most six factors that are off by EPS each, 1 - sigmoid by EPS absolutely
    out["dx"] = (lam * beta * q, eps * (WL + 6 * m) * beta * q)
    out["dgate"] = (lam * beta * x * q * (1 - q), eps * (WL + 6 * m) * beta * x.abs() * q)
    safe = torch.where(beta > 0, beta, 1.0)
    ratio = torch.where(beta > 0, a * a / safe, 0.0)
    dL = lam * (prev * a - q * x * ratio)
    dL_err = eps * (WL + 8 * m) * (mag_prev * a + q * x.abs() * ratio) + eps * m * a * W_prev
    dL_mag = m * (mag_prev * a + q * x.abs() * ratio)
    out["drate"] = (dL * L * (1 - s), (dL_err + 4 * eps * dL_mag) * L.abs())
    slope = scale * torch.sigmoid(args["decay"])
    terms, n = dL * s, float(dL.shape[0] * dL.shape[1])
    # sums of n terms: compensated over tiles, at most 64 plain additions besides
    out["ddecay"] = (-slope * terms.sum((0, 1)),
                     slope * ((dL_err + 4 * eps * dL_mag) * s).sum((0, 1))
                     + slope * (64 + n * U) * U * (dL_mag * s).sum((0, 1)))
    return out


def scan_reference(op, args, h0, dh=None, dlast=None, starts=None, scale=8.0, dtype=torch.float32):
    """args: {"a", "b"} or {"x", "rate", "gate", "decay"} on any device; results in fp64 on the CPU."""
    args = {n: t.detach().cpu().double() for n, t in args.items()}
    inputs = [n for n in args if n != "decay"]
    first = args[inputs[0]]
    H = first.shape[-1]
    states = first.shape[0] if starts is None else len(starts) - 1
    h0 = torch.zeros(states, H, dtype=torch.float64) if h0 is None else h0.detach().cpu().double()
    train = dh is not None or dlast is not None
    if train:
        dh = torch.zeros_like(first) if dh is None else dh.detach().cpu().double()
        dlast = torch.zeros_like(h0) if dlast is None else dlast.detach().cpu().double()
    if starts is None:
        tf = {n: t if n == "decay" else t.transpose(0, 1) for n, t in args.items()}
        res = _one_sequence(op, tf, h0, dh.transpose(0, 1) if train else None, dlast, scale)
        for n in list(res):
            if n in ["h"] + ["d" + i for i in inputs]:
                res[n] = tuple(v.transpose(0, 1) for v in res[n])
    else:
        per_token = ["h"] + (["d" + i for i in inputs] if train else [])
        per_state = ["state"] + (["dh0"] if train else [])
        res = {n: (torch.zeros_like(first), torch.zeros_like(first)) for n in per_token}
        res.update({n: (h0.clone() if n == "state" else dlast.clone(), torch.zeros_like(h0)) for n in per_state})
        if train and op == "gated":
            res["ddecay"] = (torch.zeros(H, dtype=torch.float64), torch.zeros(H, dtype=torch.float64))
        for n, (lo, hi) in enumerate(zip(starts[:-1], starts[1:])):
            if lo >= hi:
                continue
            part = {k: t if k == "decay" else t[lo:hi, None] for k, t in args.items()}
            one = _one_sequence(op, part, h0[n:n + 1], dh[lo:hi, None] if train else None,
                                dlast[n:n + 1] if train else None, scale)
            for k in per_token:
                for i in range(2):
                    res[k][i][lo:hi] = one[k][i][:, 0]
            for k in per_state:
                for i in range(2):
                    res[k][i][n] = one[k][i][0]
            if "ddecay" in one:
                res["ddecay"] = tuple(u + v for u, v in zip(res["ddecay"], one["ddecay"]))
    typed = ["h"] + ["d" + i for i in inputs]
    return {n: (v, e + (half_step(dtype) if n in typed else U) * v.abs() + torch.finfo(dtype).tiny)
            for n, (v, e) in res.items()}


def vocab_reference(kind, z, tau, V_threads=128, **kw):
    """Distillation (ids, teacher) or token scores (tokens); fp64 values and bounds.

    y = (z - m) / (tau ln 2) is off by 3 U |y| (difference, two roundings of the factor);
    2^y by that times ln 2 and 2 ulp; the sum of n = V / 128 + 16 additions in a row by n U of
    itself.  So log2 s is off by S = (4 U + n U) / ln 2 + 3 U E|y| with E over q, and a rounding of
    itself, log q by ln 2 (3 U |y| + S + U log2 s) + 2 U |log q|."""
    z = z.detach().cpu().double()
    V = z.shape[-1]
    live = (z > -float("inf")).any(-1, keepdim=True)
    m = z.max(-1, keepdim=True).values.masked_fill(~live, 0.0)
    w = (z - m) / tau
    logq = (w - torch.logsumexp(w, -1, keepdim=True)).masked_fill(~live, -float("inf"))
    q = logq.exp()
    ay = torch.where(q > 0, w.abs(), 0.0)
    n = V / V_threads + 16
    mean = (q * ay).sum(-1, keepdim=True)
    ls = -logq.max(-1, keepdim=True).values.masked_fill(~live, 0.0)
    S = (4 + n) * U + 3 * U * mean
    tol_log = 4 * U * w.abs() + S + 3 * U * (ls.abs() + logq.abs())
    tol_log = torch.where(logq > -float("inf"), tol_log, 0.0)
    flat = torch.where(q > 0, q * logq, 0.0)
    ent = -flat.sum(-1)
    tol_ent = (2 * (S + (4 + n) * U) * (1 + mean) + 4 * U * (q * ay * ay).sum(-1, keepdim=True)
               + 4 * U * ls.abs())[..., 0]
    return dict(logq=logq, q=q, tol_log=tol_log, ent=ent, tol_ent=tol_ent, live=live, flat=flat)


def assert_within(got, want, bound, what):
    want = torch.where(want.abs() > torch.finfo(got.dtype).max, want * float("inf"), want)  # past the type's range
    got = got.detach().cpu().double()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(want.shape)}"
    same = (got == want) | (got.isnan() & want.isnan())
    over = torch.where(same, 0.0, ((got - want).abs() - bound).nan_to_num(nan=float("inf")))
    assert bool((over <= 0).all()), (f"{what}: {int((over > 0).sum())} values past their bound, worst by "
                                     f"{over.max().item():.3e} (value {want.flatten()[over.argmax()].item():.6e}, "
                                     f"bound {bound.expand_as(want).flatten()[over.argmax()].item():.3e})")
