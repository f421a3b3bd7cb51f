"""Measured cases of the sequence operators: the linear and gated scans, the distillation
loss and the token log probabilities.

``run`` computes each operator in plain elementary torch operations (fp32, rounded once at the
end), or, with ``own`` set, through the package's public calls.  ``exact`` restates the
definitions in fp64: recurrences one token after the other, gate derivatives by autograd.

Definitions (all per channel h; t runs inside one sequence):

  linear scan   h_t = a_t h_{t-1} + b_t
  gated scan    L_t = -scale * softplus(decay) * sigmoid(rate_t),  a_t = exp(L_t),
                h_t = a_t h_{t-1} + sqrt(1 - a_t^2) * sigmoid(gate_t) * x_t
  distillation  p = softmax(teacher / tau) over the given entries (id >= 0),
                q = softmax(logits / tau) over the vocabulary,
                loss = tau^2 * sum_k p_k (log p_k - log q_{id_k})
  token scores  q as above; log q[token], entropy -sum q log q, the top-k entries of log q
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_SCALE = 8.0


def _package():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "ltc-cuda_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ltc_cuda
    return ltc_cuda


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token for each of a few sequences, at the sizes of the smallest solver configuration: pure latency
        {"name": "gated_step_small", "op": "gated_step", "dtype": "fp32", "B": 24, "H": 64},
        # one new token for a full serving batch of a wide layer
        {"name": "gated_step_wide", "op": "gated_step", "dtype": "bf16", "B": 256, "H": 4096},
        # prompts of different lengths packed without padding, a started state for each
        {"name": "gated_packed", "op": "gated_packed", "dtype": "bf16", "N": 16387, "S": 37, "H": 2048},
        # a training step of a wide layer: forward, then the gradients of inputs, decay and first state
        {"name": "gated_train", "op": "gated_train", "dtype": "bf16", "B": 8, "T": 2048, "H": 2560},
        # one very long sequence and few channels: the time axis is all the parallelism there is
        {"name": "gated_train_long", "op": "gated_train", "dtype": "fp32", "B": 1, "T": 32771, "H": 512},
        # the batch, length and width of the training configuration of the solver, gates given by the caller
        {"name": "linear_train", "op": "linear_train", "dtype": "fp32", "B": 4096, "T": 128, "H": 64},
        # a forward pass with an odd width, so that no row but the first is aligned
        {"name": "linear_odd", "op": "linear", "dtype": "fp16", "B": 3, "T": 5000, "H": 1001},
        # training on a teacher's 32 best entries for each token
        {"name": "distill_train", "op": "distill", "dtype": "bf16", "rows": 4096, "V": 32768, "K": 32, "tau": 1.0},
        # the same at an odd vocabulary in full precision, softened, with few rows
        {"name": "distill_odd", "op": "distill", "dtype": "fp32", "rows": 517, "V": 50001, "K": 8, "tau": 2.0},
        # a decoding step that reports alternatives, under a vocabulary mask
        {"name": "scores_decode", "op": "scores", "dtype": "bf16", "rows": 16, "V": 131072, "K": 8, "tau": 1.0,
         "masked": True},
        # scoring whole prompts with a few alternatives for each token, odd vocabulary
        {"name": "scores_prompt", "op": "scores", "dtype": "fp16", "rows": 8192, "V": 32003, "K": 5, "tau": 1.0,
         "masked": False},
        # a policy-gradient step: log probabilities and entropies of the sampled tokens, and their gradient
        {"name": "scores_train", "op": "scores_train", "dtype": "bf16", "rows": 4096, "V": 65536, "tau": 0.7},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["gated_step", "gated_packed", "gated_train", "gated_train", "linear", "linear_train", "distill",
                     "distill", "scores", "scores", "scores_train"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "gated_step":
        return {"op": op, "dtype": dtype, "B": _log_int(rng, 1, 512), "H": _log_int(rng, 33, 8192)}
    if op == "gated_packed":
        H = _log_int(rng, 48, 4096)
        N = _log_int(rng, 64, max(64, min(65536, 32_000_000 // H)))
        return {"op": op, "dtype": dtype, "N": N, "S": _log_int(rng, 1, max(1, min(200, N // 4))), "H": H}
    if op in ("gated_train", "linear", "linear_train"):
        H = _log_int(rng, 17, 4096)
        T = _log_int(rng, 2, 32768)
        B = _log_int(rng, 1, max(1, min(4096, 32_000_000 // (H * T))))
        return {"op": op, "dtype": dtype, "B": B, "T": T, "H": H}
    V = _log_int(rng, 1000, 160_000)
    rows = _log_int(rng, 1, max(1, min(16384, 130_000_000 // V)))
    tau = rng.choice([1.0, 0.5, 0.8, 2.0])
    if op == "distill":
        return {"op": op, "dtype": dtype, "rows": rows, "V": V, "K": _log_int(rng, 1, 128), "tau": tau}
    if op == "scores":
        return {"op": op, "dtype": dtype, "rows": rows, "V": V, "K": rng.randint(0, 20), "tau": tau,
                "masked": rng.random() < 0.5}
    return {"op": op, "dtype": dtype, "rows": rows, "V": V, "tau": tau}


def work(case):
    op, e = case["op"], _BYTES[case["dtype"]]
    if op == "gated_step":
        n = case["B"] * case["H"]
        return {"bytes": n * (4 * e + 8) + 4 * case["H"], "flops": 20 * n}
    if op == "gated_packed":
        n, s = case["N"] * case["H"], case["S"] * case["H"]
        return {"bytes": n * 4 * e + 8 * s + 4 * case["H"] + 4 * (case["S"] + 1), "flops": 20 * n}
    if op in ("gated_train", "linear", "linear_train"):
        n, s = case["B"] * case["T"] * case["H"], case["B"] * case["H"]
        if op == "linear":
            return {"bytes": n * 3 * e + 8 * s, "flops": 2 * n}
        if op == "linear_train":  # a, b, dL/dh read; h, da, db written; h0, its gradient, both ends of the final state
            return {"bytes": n * 6 * e + 16 * s, "flops": 5 * n}
        return {"bytes": n * 8 * e + 16 * s + 8 * case["H"], "flops": 60 * n}
    n, r = case["rows"] * case["V"], case["rows"]
    if op == "distill":
        return {"bytes": 2 * n * e + r * (case["K"] * (8 + e) + 8), "flops": 7 * n}
    if op == "scores":
        return {"bytes": n * e + r * (8 + 8 + 12 * case["K"]), "flops": 6 * n}
    return {"bytes": 2 * n * e + r * (8 + 16), "flops": 12 * n}


# ---------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, op = _TYPES[case["dtype"]], case["op"]

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).add_(shift)

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=g, device="cuda").mul_(hi - lo).add_(lo)

    s = {"op": op, "case": dict(case)}
    if op.startswith("gated"):
        H = case["H"]
        lead = {"gated_step": (case.get("B"),), "gated_packed": (case.get("N"),)}.get(op) or (case["B"], case["T"])
        s["x"] = normal(*lead, H).to(dt)
        s["rate"] = normal(*lead, H, scale=1.5).to(dt)
        s["gate"] = normal(*lead, H, scale=1.5).to(dt)
        # decay such that a = exp(-scale * softplus(decay)) spreads over (0.9, 0.999) at an open gate
        s["decay"] = torch.log(torch.expm1(-torch.log(uniform(0.9, 0.999, H)) / _SCALE * 2))
        states = case["S"] if op == "gated_packed" else case["B"]
        s["h0"] = normal(states, H, scale=0.5)
        if op == "gated_packed":
            cuts = torch.sort(torch.randint(0, case["N"] + 1, (case["S"] - 1,), generator=g, device="cuda")).values
            tail = max(0, min(5, case["N"] - 64))  # a few unused rows behind the last sequence
            ends = torch.cat([torch.zeros(1, device="cuda"), cuts, torch.full((1,), case["N"], device="cuda")])
            s["seq_starts"] = ends.clamp(max=case["N"] - tail).to(torch.int32)
        if op == "gated_train":
            s["dh"] = normal(*lead, H).to(dt)
            s["dlast"] = normal(case["B"], H)
    elif op.startswith("linear"):
        B, T, H = case["B"], case["T"], case["H"]
        s["a"] = torch.exp(-uniform(0.001, 0.5, B, T, H)).to(dt)
        s["b"] = normal(B, T, H, scale=0.3).to(dt)
        s["h0"] = normal(B, H, scale=0.5)
        if op == "linear_train":
            s["dh"] = normal(B, T, H).to(dt)
            s["dlast"] = normal(B, H)
    else:
        rows, V = case["rows"], case["V"]
        z = normal(rows, V, scale=2.5)
        s["tau"] = float(case["tau"])
        if op == "distill":
            K = min(case["K"], V)
            near = (z + normal(rows, V)).topk(K, dim=1)
            s["teacher_ids"] = near.indices
            s["teacher"] = (near.values * 1.3).to(dt)
            # some rows have fewer entries, and one in 64 none at all (a position outside the loss)
            s["teacher_ids"][::7, K - K // 4:] = -1
            s["teacher_ids"][5::64] = -1
            s["dloss"] = uniform(0.5, 1.5, rows) / rows
        else:
            s["tokens"] = torch.randint(0, V, (rows,), generator=g, device="cuda")
            s["tokens"][::2] = z[::2].argmax(dim=1)
            if rows > 8:
                s["tokens"][3::37] = -1  # positions outside the score
            if case.get("masked"):
                z.masked_fill_(uniform(0, 1, V) < 0.3, -math.inf)
                if rows > 4:
                    z[4] = -math.inf  # a mask that leaves nothing
            if op == "scores_train":
                s["dlogprob"] = normal(rows) / rows
                s["dentropy"] = torch.full((rows,), 0.01 / rows, device="cuda")
        s["logits"] = z.to(dt)
    return s


# ---------------------------------------------------------------------------- plain form
def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim -2 with h_{-1} = 0, in log2(T) doubling steps."""
    T, k = a.shape[-2], 1
    while k < T:
        b = torch.cat([b[..., :k, :], b[..., k:, :] + a[..., k:, :] * b[..., :-k, :]], dim=-2)
        a = torch.cat([a[..., :k, :], a[..., k:, :] * a[..., :-k, :]], dim=-2)
        k *= 2
    return b


def _gates(s):
    x, rate, gate = s["x"].float(), torch.sigmoid(s["rate"].float()), torch.sigmoid(s["gate"].float())
    L = -_SCALE * torch.log1p(torch.exp(s["decay"])) * rate
    return x, rate, gate, L, torch.exp(L), torch.sqrt(-torch.expm1(2 * L))


def _with_first(a, b, h0):
    """The given first state folded into the first token: a h0 + b, and a = 0 there."""
    b = torch.cat([b[:, :1] + a[:, :1] * h0[:, None], b[:, 1:]], dim=1)
    return torch.cat([torch.zeros_like(a[:, :1]), a[:, 1:]], dim=1), b


def _adjoint(a, dh, dlast):
    """lambda_t = dh_t + a_{t+1} lambda_{t+1}, the last one with the final state's gradient."""
    dh = torch.cat([dh[:, :-1], dh[:, -1:] + dlast[:, None]], dim=1)
    nxt = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], dim=1)
    return _scan(nxt.flip(1), dh.flip(1)).flip(1)


def _plain_scan(s):
    op = s["op"]
    if op.startswith("linear"):
        dt, a, b = s["a"].dtype, s["a"].float(), s["b"].float()
    else:
        dt = s["x"].dtype
        x, rate, gate, L, a, beta = _gates(s)
        b = beta * gate * x
    if op == "gated_step":
        h = a * s["h0"] + b
        return {"h": h.to(dt), "state": h}
    if op == "gated_packed":
        starts = s["seq_starts"].long()
        lo, hi = starts[:-1], starts[1:]
        live = lo < hi
        at = torch.arange(a.shape[0], device=a.device)
        inside = ((at >= starts[0]) & (at < starts[-1]))[:, None]
        first, h0 = lo[live], s["h0"][live]
        b = b.index_put((first,), b[first] + a[first] * h0)
        a = a.index_put((first,), torch.zeros_like(h0))
        h = torch.where(inside, _scan(a, b), 0.0)
        last = torch.where(live[:, None], h[(hi - 1).clamp(min=0)], s["h0"])
        return {"h": h.to(dt), "state": last}
    h = _scan(*_with_first(a, b, s["h0"]))
    out = {"h": h.to(dt), "state": h[:, -1].clone()}
    if op == "linear":
        return out
    lam = _adjoint(a, s["dh"].float(), s["dlast"])
    prev = torch.cat([s["h0"][:, None], h[:, :-1]], dim=1)
    out["dh0"] = a[:, 0] * lam[:, 0]
    if op == "linear_train":
        return {**out, "da": (lam * prev).to(dt), "db": lam.to(dt)}
    out["dx"] = (lam * beta * gate).to(dt)
    out["dgate"] = (lam * beta * x * gate * (1 - gate)).to(dt)
    open_ = beta > 0
    dL = lam * prev * a - torch.where(open_, lam * gate * x * a * a / torch.where(open_, beta, 1.0), 0.0)
    out["drate"] = (dL * L * (1 - rate)).to(dt)
    out["ddecay"] = (dL * rate).double().sum(dim=(0, 1)).float() * (-_SCALE * torch.sigmoid(s["decay"]))
    return out


def _log_softmax(z, tau):
    """log softmax(z / tau) over the last dimension, -inf everywhere in a row with nothing but -inf."""
    top = z.max(dim=-1, keepdim=True).values
    empty = top == -math.inf
    y = (z - torch.where(empty, 0.0, top)) / tau
    total = torch.exp(y).sum(dim=-1, keepdim=True)
    return y - torch.where(empty, 0.0, torch.log(total))


def _plain_logits(s):
    z, tau, op = s["logits"].float(), s["tau"], s["op"]
    logq = _log_softmax(z, tau)
    q = torch.exp(logq)
    if op == "distill":
        ids, there = s["teacher_ids"].clamp(min=0), s["teacher_ids"] >= 0
        logp = _log_softmax(torch.where(there, s["teacher"].float(), -math.inf), tau)
        p = torch.exp(logp)
        loss = tau * tau * torch.where(p > 0, p * (logp - logq.gather(1, ids)), 0.0).sum(dim=1)
        has = there.any(dim=1, keepdim=True)
        dz = torch.where(has, q, 0.0).scatter_add(1, ids, -p) * (tau * s["dloss"])[:, None]
        return {"loss": loss, "dlogits": dz.to(s["logits"].dtype)}
    there = s["tokens"] >= 0
    tok = s["tokens"].clamp(min=0)[:, None]
    entropy = -torch.where(q > 0, q * logq, 0.0).sum(dim=1)
    out = {"logprob": torch.where(there, logq.gather(1, tok)[:, 0], 0.0), "entropy": entropy}
    if op == "scores":
        k = s["case"]["K"]
        if k:
            best = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
            top = logq.gather(1, best)
            out["top_ids"], out["top_logprobs"] = torch.where(top > -math.inf, best, -1), top
        return out
    dlp = torch.where(there, s["dlogprob"], 0.0)[:, None]
    slope = torch.where(q > 0, q * (logq + entropy[:, None]), 0.0)
    dz = (-q * dlp).scatter_add(1, tok, dlp) - slope * s["dentropy"][:, None]
    return {**out, "dlogits": (dz / tau).to(s["logits"].dtype)}


# ---------------------------------------------------------------------------- the package's operators
def _own(s):
    ltc = _package()
    op = s["op"]
    if op == "gated_step":
        h, state = ltc.ltc_gated_scan_step(s["x"], s["rate"], s["gate"], s["decay"], s["h0"], scale=_SCALE)
        return {"h": h, "state": state}
    if op == "gated_packed":
        with torch.no_grad():
            h, state = ltc.ltc_gated_scan(s["x"], s["rate"], s["gate"], s["decay"], s["h0"],
                                          seq_starts=s["seq_starts"], scale=_SCALE)
        return {"h": h, "state": state}
    if op == "linear":
        with torch.no_grad():
            h, state = ltc.ltc_linear_scan(s["a"], s["b"], s["h0"])
        return {"h": h, "state": state}
    if op in ("linear_train", "gated_train"):
        names = ("a", "b", "h0") if op == "linear_train" else ("x", "rate", "gate", "decay", "h0")
        leaves = [s[n].detach().requires_grad_(True) for n in names]
        h, state = ltc.ltc_linear_scan(*leaves) if op == "linear_train" else ltc.ltc_gated_scan(*leaves, scale=_SCALE)
        grads = torch.autograd.grad([h, state], leaves, [s["dh"], s["dlast"]])
        return {"h": h.detach(), "state": state.detach(), **{"d" + n: v for n, v in zip(names, grads)}}
    if op == "scores":
        with torch.no_grad():
            r = ltc.ltc_token_logprobs(s["logits"], s["tokens"], top_k=s["case"]["K"], temperature=s["tau"])
        out = {"logprob": r.logprobs, "entropy": r.entropy}
        return {**out, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs} if s["case"]["K"] else out
    z = s["logits"].detach().requires_grad_(True)
    if op == "distill":
        loss = ltc.ltc_distill_loss(z, s["teacher_ids"], s["teacher"], temperature=s["tau"])
        (dz,) = torch.autograd.grad([loss], [z], [s["dloss"]])
        return {"loss": loss.detach(), "dlogits": dz}
    r = ltc.ltc_token_logprobs(z, s["tokens"], temperature=s["tau"])
    (dz,) = torch.autograd.grad([r.logprobs, r.entropy], [z], [s["dlogprob"], s["dentropy"]])
    return {"logprob": r.logprobs.detach(), "entropy": r.entropy.detach(), "dlogits": dz}


def run(state):
    if own:
        return _own(state)
    return _plain_scan(state) if "h0" in state else _plain_logits(state)


# ---------------------------------------------------------------------------- fp64 definitions
def _walk(a, b, h):
    """All states of one batch of sequences, one token after the other (fp64; time first)."""
    out = torch.empty_like(b)
    for t in range(a.shape[0]):
        h = torch.addcmul(b[t], a[t], h, out=out[t])
    return out


def _exact_scan(s):
    op = s["op"]
    names = ("a", "b") if op.startswith("linear") else ("x", "rate", "gate", "decay")
    train = op.endswith("train")
    leaf = {n: s[n].double().requires_grad_(train) for n in names}
    if op.startswith("linear"):
        a, b = leaf["a"], leaf["b"]
    else:
        log_a = _SCALE * torch.nn.functional.logsigmoid(-leaf["decay"]) / (1 + torch.exp(-leaf["rate"]))
        a = log_a.exp()
        b = (1 - (2 * log_a).exp()).sqrt() * leaf["x"] / (1 + torch.exp(-leaf["gate"]))
    h0 = s["h0"].double()
    with torch.no_grad():
        if op == "gated_step":
            h = a * h0 + b
            return {"h": h, "state": h}
        if op == "gated_packed":
            ends = s["seq_starts"].tolist()
            h, last = torch.zeros_like(b), h0.clone()
            for n, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
                if lo < hi:
                    h[lo:hi] = _walk(a[lo:hi], b[lo:hi], h0[n])
                    last[n] = h[hi - 1]
            return {"h": h, "state": last}
        at, bt = a.transpose(0, 1).contiguous(), b.transpose(0, 1).contiguous()
        h = _walk(at, bt, h0)
        out = {"h": h.transpose(0, 1), "state": h[-1].clone()}
        if not train:
            return out
        lam = torch.empty_like(h)
        carry = s["dlast"].double()
        dh = s["dh"].transpose(0, 1).double()
        for t in range(h.shape[0] - 1, -1, -1):
            lam[t] = dh[t] + carry
            carry = at[t] * lam[t]
        out["dh0"] = carry
        prev = torch.cat([h0[None], h[:-1]])
        da, db = (lam * prev).transpose(0, 1), lam.transpose(0, 1)
    grads = torch.autograd.grad([a, b], [leaf[n] for n in names], [da, db])
    return {**out, **{"d" + n: v for n, v in zip(names, grads)}}


def _exact_row_block(s, lo, hi):
    op, tau = s["op"], s["tau"]
    z = s["logits"][lo:hi].double()
    live = (z > -math.inf).any(dim=1, keepdim=True)
    w = (z / tau).masked_fill(~live, 0.0)
    logq = (w - torch.logsumexp(w, dim=1, keepdim=True)).masked_fill(~live, -math.inf)
    q = logq.exp()
    hot = torch.zeros_like(q)
    if op == "distill":
        ids = s["teacher_ids"][lo:hi]
        t = (s["teacher"][lo:hi].double() / tau).masked_fill(ids < 0, -math.inf)
        has = (ids >= 0).any(dim=1, keepdim=True)
        p = torch.softmax(t.masked_fill(~has, 0.0), dim=1) * has
        each = torch.special.xlogy(p, p) - torch.where(p > 0, p * logq.gather(1, ids.clamp(min=0)), 0.0)
        hot.scatter_add_(1, ids.clamp(min=0), p)
        grad = (q * has - hot) * tau * s["dloss"][lo:hi, None].double()
        return {"loss": tau ** 2 * each.sum(dim=1), "dlogits": grad}
    tok = s["tokens"][lo:hi]
    lp = logq.gather(1, tok.clamp(min=0)[:, None])[:, 0].masked_fill(tok < 0, 0.0)
    entropy = torch.special.entr(q).sum(dim=1)
    out = {"logprob": lp, "entropy": entropy}
    if op == "scores":
        if s["case"]["K"]:
            out["top_ids"], out["top_logprobs"] = None, logq.sort(dim=1, descending=True).values[:, :s["case"]["K"]]
        return out
    hot.scatter_(1, tok.clamp(min=0)[:, None], 1.0)
    dlp = s["dlogprob"][lo:hi].double().masked_fill(tok < 0, 0.0)[:, None]
    dent = s["dentropy"][lo:hi].double()[:, None]
    grad = (dlp * (hot - q) + dent * (torch.special.entr(q) - q * entropy[:, None])) / tau
    return {**out, "dlogits": grad}


def exact(case, seed):
    s = prepare(case, seed)
    if "h0" in s:
        return _exact_scan(s)
    step = max(1, 40_000_000 // case["V"])
    blocks = [_exact_row_block(s, lo, min(lo + step, case["rows"])) for lo in range(0, case["rows"], step)]
    return {n: None if blocks[0][n] is None else torch.cat([b[n] for b in blocks]) for n in blocks[0]}
