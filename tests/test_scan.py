"""GPU: ltc_linear_scan, ltc_gated_scan and ltc_gated_scan_step against the fp64 recurrence."""
import ctypes

import pytest
import torch

import ltc_cuda
from sequence_ref import assert_within, half_step, scan_reference

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(op, lead, H, dtype, seed, states, h0=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    if op == "linear":
        args = {"a": torch.rand(*lead, H, generator=g) * 1.2 - 0.2, "b": r(*lead, H)}
    else:
        args = {"x": r(*lead, H), "rate": r(*lead, H).clamp(-4, 4) * 1.5, "gate": r(*lead, H).clamp(-4, 4) * 1.5}
    args = {n: t.to(dtype).cuda() for n, t in args.items()}
    if op == "gated":
        args["decay"] = (r(H) - 3).cuda()
    return (args, r(states, H).cuda() if h0 else None, r(*lead, H).to(dtype).cuda(), r(states, H).cuda())


def call(op, args, h0, starts=None):
    fn = ltc_cuda.ltc_linear_scan if op == "linear" else ltc_cuda.ltc_gated_scan
    return fn(*args.values(), h0, seq_starts=starts)


def check(op, args, h0, dh, dlast, dtype, starts=None, what=""):
    leaves = {n: t.detach().requires_grad_(True) for n, t in args.items()}
    lh0 = None if h0 is None else h0.detach().requires_grad_(True)
    dev_starts = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
    h, last = call(op, leaves, lh0, dev_starts)
    assert h.dtype == dtype and last.dtype == torch.float32
    wrt = list(leaves.values()) + ([] if h0 is None else [lh0])
    grads = torch.autograd.grad([h, last], wrt, [dh, dlast])
    got = {"h": h, "state": last, **{"d" + n: g for n, g in zip([*leaves, "h0"], grads)}}
    ref = scan_reference(op, args, h0, dh, dlast, starts, dtype=dtype)
    for n, v in got.items():
        assert_within(v, *ref[n], f"{what} {n}")
    with torch.no_grad():  # a forward without a backward gives the same bits
        h2, last2 = call(op, args, h0, dev_starts)
    assert torch.equal(h2, h) and torch.equal(last2, last)


SHAPES = [(1, 1, 1), (3, 2, 4), (2, 15, 33), (5, 16, 8), (2, 17, 64), (1, 63, 36), (2, 64, 12), (1, 65, 5),
          (3, 130, 100), (2, 257, 40)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("op", ["linear", "gated"])
@pytest.mark.parametrize("B,T,H", SHAPES)
def test_padded(op, B, T, H, dtype):
    args, h0, dh, dlast = make(op, (B, T), H, dtype, B * 1000 + T * 10 + H, B, h0=(B + T) % 3 != 0)
    check(op, args, h0, dh, dlast, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("op", ["linear", "gated"])
@pytest.mark.parametrize("B,T,H", [(1, 1500, 8), (1, 1500, 7), (1, 2300, 40), (3, 700, 600), (2, 400, 1301)])
def test_clusters(op, B, T, H, dtype):
    """Few chains: a cluster of blocks takes each, in narrow items where there are fewest."""
    dims = ltc_cuda.LtcScanDims(B, T, H, 0, 0)
    p = ltc_cuda.LtcScanPlan()
    assert ltc_cuda._lib.ltc_scan_plan(ctypes.byref(dims), ctypes.byref(p)) == 0 and p.cluster > 1
    args, h0, dh, dlast = make(op, (B, T), H, dtype, H, B)
    check(op, args, h0, dh, dlast, dtype)


PACKED = [([0, 5], 5), ([0, 0, 1, 1, 4, 70, 70], 73), ([0, 64, 128, 129], 129), ([0, 1, 2, 3, 3, 200], 210),
          ([0, 700, 1300], 1300), ([3, 9], 12), ([0, 0], 4)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("op", ["linear", "gated"])
@pytest.mark.parametrize("starts,N", PACKED)
@pytest.mark.parametrize("H", [12, 5])
def test_packed(op, starts, N, H, dtype):
    args, h0, dh, dlast = make(op, (N,), H, dtype, N + H, len(starts) - 1, h0=N % 2 == 1)
    check(op, args, h0, dh, dlast, dtype, starts)


@pytest.mark.parametrize("op", ["linear", "gated"])
@pytest.mark.parametrize("long", [False, True])
def test_packed_sequences_are_isolated(op, long):
    """Whatever lies outside the sequences, and infinities and NaN in one sequence, stay there."""
    starts, N, H = ([2, 40, 90, 97], 100, 8) if not long else ([2, 900, 1700, 1990], 2000, 8)
    args, h0, dh, dlast = make(op, (N,), H, torch.float32, 5, 3)
    t = torch.tensor(starts, dtype=torch.int32, device="cuda")

    def run(a, d):
        leaves = [v.detach().requires_grad_(True) for v in a.values()]
        h, last = call(op, dict(zip(a, leaves)), h0, t)
        grads = torch.autograd.grad([h, last], leaves, [d, dlast])
        return h.detach(), last.detach(), grads

    clean = run(args, dh)
    dirty = {n: v.clone() for n, v in args.items()}
    d2 = dh.clone()
    for n, v in dirty.items():
        if n != "decay":
            v[:2] = float("nan")
            v[starts[3]:] = float("inf")
            v[starts[1] + 3] = float("nan")   # inside the second sequence
    first = "a" if op == "linear" else "x"
    dirty[first][starts[1] + 1] = float("inf")
    d2[:2], d2[starts[3]:] = float("nan"), float("nan")
    got = run(dirty, d2)
    for lo, hi in ((0, starts[1]), (starts[2], N)):
        assert torch.equal(got[0][lo:hi], clean[0][lo:hi])
        for n, g, c in zip(args, got[2], clean[2]):
            if n != "decay":
                assert torch.equal(g[lo:hi], c[lo:hi]), n
    assert torch.equal(got[1][[0, 2]], clean[1][[0, 2]]) and got[1][1].isnan().all()
    assert (got[0][:2] == 0).all() and (got[0][starts[3]:] == 0).all()
    for g in got[2][:2]:
        assert (g[:2] == 0).all() and (g[starts[3]:] == 0).all()


@pytest.mark.parametrize("op", ["linear", "gated"])
def test_a_channel_and_a_row_do_not_leak(op):
    args, h0, dh, dlast = make(op, (3, 70), 12, torch.float32, 9, 3)
    h, last = call(op, args, h0)
    bad = {n: v.clone() for n, v in args.items()}
    bad["b" if op == "linear" else "x"][1, 4, 5] = float("nan")
    hb, lb = call(op, bad, h0)
    assert hb[1, 4:, 5].isnan().all() and lb[1, 5].isnan()
    hb[1, 4:, 5], lb[1, 5] = h[1, 4:, 5], last[1, 5]
    assert torch.equal(hb, h) and torch.equal(lb, last)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_strided_inputs(dtype):
    """Slices of one projection, time-major storage, a broadcast gate, a summed output."""
    B, T, H = 3, 70, 20
    args, h0, dh, dlast = make("gated", (B, T), H, dtype, 3, B)
    want = call("gated", args, h0)
    joint = torch.cat([args["x"], args["rate"], args["gate"]], dim=-1)
    x, rate, gate = joint.split(H, dim=-1)
    got = ltc_cuda.ltc_gated_scan(x, rate, gate, args["decay"], h0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    off = torch.empty(B, T, 3 * H + 1, dtype=dtype, device="cuda")[..., 1:]  # rows that start off 16 bytes
    off.copy_(joint)
    x, rate, gate = off.split(H, dim=-1)
    got = ltc_cuda.ltc_gated_scan(x, rate, gate, args["decay"], h0)
    assert torch.allclose(got[0].float(), want[0].float(), rtol=4 * half_step(dtype), atol=1e-5)
    tm = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in list(args.values())[:3]]
    got = ltc_cuda.ltc_gated_scan(*tm, args["decay"], h0)
    assert torch.equal(got[0], want[0])
    # a broadcast along time and batch; the gradient of the broadcast tensor is the sum
    a = torch.rand(1, 1, H, device="cuda").to(dtype).requires_grad_(True)
    b = args["x"].detach().requires_grad_(True)
    h, last = ltc_cuda.ltc_linear_scan(a.expand(B, T, H), b, h0)
    da, db = torch.autograd.grad(h.sum(), [a, b])
    ref = scan_reference("linear", {"a": a.expand(B, T, H), "b": b}, h0, torch.ones_like(h), None, dtype=dtype)
    assert_within(db, *ref["db"], "db")
    # the sum over B*T rounded entries, itself rounded to the type
    v, e = ref["da"]
    assert_within(da, v.sum((0, 1), keepdim=True),
                  e.sum((0, 1), keepdim=True) + 4 * half_step(dtype) * v.abs().sum((0, 1), keepdim=True), "da")


def test_last_dim_strided_is_copied():
    a = torch.rand(2, 8, 30, device="cuda")
    b = torch.randn(2, 8, 30, device="cuda")
    h, last = ltc_cuda.ltc_linear_scan(a.transpose(1, 2), b.transpose(1, 2))
    want, wl = ltc_cuda.ltc_linear_scan(a.transpose(1, 2).contiguous(), b.transpose(1, 2).contiguous())
    assert torch.equal(h, want) and torch.equal(last, wl)


@pytest.mark.parametrize("only", ["h", "state"])
@pytest.mark.parametrize("op", ["linear", "gated"])
def test_one_incoming_gradient(op, only):
    args, h0, dh, dlast = make(op, (2, 80), 8, torch.float32, 4, 2)
    leaves = {n: t.detach().requires_grad_(True) for n, t in args.items()}
    h, last = call(op, leaves, None)
    out, g = (h, dh) if only == "h" else (last, dlast)
    grads = torch.autograd.grad([out], list(leaves.values()), [g])
    ref = scan_reference(op, args, None, dh if only == "h" else None, dlast if only == "state" else None)
    for n, v in zip(leaves, grads):
        assert_within(v, *ref["d" + n], n)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,H", [(1, 1), (7, 33), (24, 64), (3, 100)])
def test_step(B, H, dtype):
    args, h0, _, _ = make("gated", (B, 1), H, dtype, B + H, B)
    flat = [t[:, 0] if n != "decay" else t for n, t in args.items()]
    want, wl = call("gated", args, h0)
    h, s = ltc_cuda.ltc_gated_scan_step(*flat, h0)
    assert torch.equal(h, want[:, 0]) and torch.equal(s, wl)
    state = h0.clone()
    h2, s2 = ltc_cuda.ltc_gated_scan_step(*flat, state, out_state=state)
    assert s2 is state and torch.equal(state, s) and torch.equal(h2, h)
    joint = torch.cat([flat[0], flat[1], flat[2]], dim=1).split(H, dim=1)
    h3, s3 = ltc_cuda.ltc_gated_scan_step(*joint, flat[3], h0)
    assert torch.allclose(s3, s, rtol=1e-5, atol=1e-6)


def test_steps_continue_a_scan():
    args, h0, _, _ = make("gated", (2, 40), 24, torch.float32, 8, 2)
    want, wl = call("gated", args, h0)
    state, seen = h0.clone(), []
    for t in range(40):
        h, _ = ltc_cuda.ltc_gated_scan_step(args["x"][:, t], args["rate"][:, t], args["gate"][:, t], args["decay"],
                                            state, out_state=state)
        seen.append(h)
    ref = scan_reference("gated", args, h0)
    assert_within(torch.stack(seen, 1), *ref["h"], "h")
    assert_within(state, *ref["state"], "state")
    # and a scan in two pieces is the scan
    h1, s1 = call("gated", {n: t if n == "decay" else t[:, :23] for n, t in args.items()}, h0)
    h2, s2 = call("gated", {n: t if n == "decay" else t[:, 23:] for n, t in args.items()}, s1)
    assert_within(torch.cat([h1, h2], 1), *ref["h"], "pieces")
    assert_within(s2, *ref["state"], "pieces' state")


def test_saturated_gates():
    """Open, shut and vanishing gates: a = 1 exactly, a = 0, and gradients that stay finite."""
    H = 8
    rate = torch.tensor([-200.0, -90.0, -30.0, 0.0, 30.0, 90.0, 200.0, -15.0], device="cuda").expand(2, 70, H)
    gate = rate.flip(-1)
    decay = torch.tensor([-100.0, -20.0, -3.0, 0.0, 3.0, 20.0, 50.0, -60.0], device="cuda")
    for perm in range(H):
        d = decay.roll(perm).clone().requires_grad_(True)
        x = torch.randn(2, 70, H, device="cuda", requires_grad=True)
        r, q = rate.clone().requires_grad_(True), gate.clone().requires_grad_(True)
        h, last = ltc_cuda.ltc_gated_scan(x, r, q, d)
        grads = torch.autograd.grad(h.sum() + last.sum(), [x, r, q, d])
        for v in (h, last, *grads):
            assert torch.isfinite(v).all()
        L = -8.0 * torch.nn.functional.softplus(d.double(), threshold=1000) * torch.sigmoid(rate.double())
        a, b = L.exp(), (-torch.expm1(2 * L)).sqrt() * torch.sigmoid(gate.double()) * x.double()
        want = torch.zeros(2, H, device="cuda", dtype=torch.float64)
        for t in range(70):
            want = a[:, t] * want + b[:, t]
        assert torch.allclose(last.double(), want, rtol=2e-4, atol=1e-5)


@pytest.mark.parametrize("op", ["linear", "gated"])
def test_gradient_against_differences(op):
    """Directional derivatives of the fp64 recurrence, central differences of step 1e-4
    (error of second order: 1e-8 of the third derivative's scale, 1e-6 allowed)."""
    args, h0, dh, dlast = make(op, (2, 90), 6, torch.float32, 12, 2)
    leaves = {n: t.detach().requires_grad_(True) for n, t in args.items()}
    h, last = call(op, leaves, h0)
    grads = torch.autograd.grad([h, last], list(leaves.values()), [dh, dlast])

    def loss(a):
        r = scan_reference(op, a, h0)
        return (r["h"][0] * dh.cpu().double()).sum() + (r["state"][0] * dlast.cpu().double()).sum()

    for (n, t), g in zip(args.items(), grads):
        d = torch.randn(t.shape, generator=torch.Generator().manual_seed(1)).double()
        up, dn = ({**args, n: t.cpu().double() + e * d} for e in (1e-4, -1e-4))
        slope = ((loss(up) - loss(dn)) / 2e-4).item()
        mine = (g.cpu().double() * d).sum().item()
        assert abs(slope - mine) <= 1e-5 * max(1.0, (g.cpu().double() * d).abs().sum().item()), n


def test_deterministic_and_independent_of_the_batch():
    for op in ("linear", "gated"):
        for lead, H in (((4, 300), 36), ((70, 9), 36)):
            args, h0, dh, dlast = make(op, lead, H, torch.float32, 2, lead[0])
            runs = []
            for _ in range(2):
                leaves = [t.detach().requires_grad_(True) for t in args.values()]
                h, last = call(op, dict(zip(args, leaves)), h0)
                runs.append([h, last, *torch.autograd.grad([h, last], leaves, [dh, dlast])])
            for u, v in zip(*runs):
                assert torch.equal(u, v)


def test_empty():
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    h0 = torch.randn(2, 3, device="cuda").requires_grad_(True)
    h, last = ltc_cuda.ltc_linear_scan(z(2, 0, 3), z(2, 0, 3), h0)
    assert h.shape == (2, 0, 3) and torch.equal(last, h0)
    assert torch.equal(torch.autograd.grad(last.sum(), h0)[0], torch.ones_like(h0))
    assert ltc_cuda.ltc_gated_scan(z(0, 4, 3), z(0, 4, 3), z(0, 4, 3), z(3))[1].shape == (0, 3)
    starts = torch.zeros(3, dtype=torch.int64, device="cuda")
    assert torch.equal(ltc_cuda.ltc_linear_scan(z(0, 3), z(0, 3), h0.detach(), starts)[1], h0)
    assert ltc_cuda.ltc_gated_scan_step(z(0, 3), z(0, 3), z(0, 3), z(3), z(0, 3))[0].shape == (0, 3)


def test_offsets_past_32_bits():
    """2^31 elements and more: the last rows against the recurrence from a reset in front of them."""
    T, H = (1 << 20) + 5, 2050
    a = torch.full((1, 1, H), 0.5, device="cuda", dtype=torch.float16).expand(1, T, H)
    b = torch.zeros(1, T, H, device="cuda", dtype=torch.float16)
    tail = torch.randn(40, H, device="cuda").half()
    b[0, -40:] = tail
    with torch.no_grad():
        h, last = ltc_cuda.ltc_linear_scan(a, b)
    ref = scan_reference("linear", {"a": torch.full((1, 40, H), 0.5), "b": tail[None]}, None, dtype=torch.float16)
    assert_within(h[:, -40:], *ref["h"], "h")
    assert_within(last, *ref["state"], "state")
    assert bool((h[0, :-40] == 0).all())


def test_streams_and_graphs():
    """A side stream, and a captured forward and backward replayed on new inputs."""
    args, h0, dh, dlast = make("gated", (3, 200), 24, torch.float32, 21, 3)
    new, h0b, dhb, dlb = make("gated", (3, 200), 24, torch.float32, 22, 3)

    def step(a, s, g, gl):
        leaves = [t.detach().requires_grad_(True) for t in a.values()]
        h, last = call("gated", dict(zip(a, leaves)), s)
        return [h.detach(), last.detach(), *torch.autograd.grad([h, last], leaves, [g, gl])]

    want = step(new, h0b, dhb, dlb)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(new, h0b, dhb, dlb)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u, v) for u, v in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(args, h0, dh, dlast)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step(args, h0, dh, dlast)
    for t, n in zip([*args.values(), h0, dh, dlast], [*new.values(), h0b, dhb, dlb]):
        t.copy_(n)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(out, want))


def test_captured_cluster_of_sixteen():
    """The largest cluster (a launch attribute beyond the portable size), captured and replayed
    twice on changed inputs, padded and packed."""
    args, h0, dh, dlast = make("gated", (1, 4200), 16, torch.bfloat16, 31, 1)
    new = make("gated", (1, 4200), 16, torch.bfloat16, 32, 1)
    starts = torch.tensor([0, 100, 100, 4100], dtype=torch.int32, device="cuda")

    def step(a, g, gl):
        leaves = [t.detach().requires_grad_(True) for t in a.values()]
        h, last = call("gated", dict(zip(a, leaves)), None)
        flat = {n: t if n == "decay" else t[0] for n, t in zip(a, leaves)}
        hp, lp = call("gated", flat, None, starts)
        return [h.detach(), hp.detach(), lp.detach(), *torch.autograd.grad([h, last, hp], leaves, [g, gl, g[0]])]

    step(args, dh, dlast)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(args, dh, dlast)
    for t, n in zip([*args.values(), dh, dlast], [*new[0].values(), new[2], new[3]]):
        t.copy_(n)
    want = step(new[0], new[2], new[3])
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(out, want))


def test_two_streams_at_once():
    """Two scans in flight on two streams share nothing."""
    jobs = [make(op, (2, 3000), 20, torch.float32, i, 2) for i, op in enumerate(("linear", "gated"))]
    want = [call(op, j[0], j[1]) for op, j in zip(("linear", "gated"), jobs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = []
    for _ in range(3):
        for op, j, st in zip(("linear", "gated"), jobs, streams):
            with torch.cuda.stream(st):
                got.append(call(op, j[0], j[1]))
    torch.cuda.synchronize()
    for i, (h, last) in enumerate(got):
        assert torch.equal(h, want[i % 2][0]) and torch.equal(last, want[i % 2][1])


def test_solver_without_recurrent_synapses_is_a_linear_scan():
    """With w_pos = 0 an unfold is v <- (cm v + gleak vleak + num) / (cm + gleak + den + eps):
    for one unfold a step, the scan over a = cm / (...), b = (gleak vleak + num) / (...)."""
    B, T, D, H, eps = 3, 50, 7, 20, 1e-8
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.rand(*s, generator=g).cuda()  # noqa: E731
    x, h0 = torch.randn(B, T, D, generator=g).cuda(), torch.randn(B, H, generator=g).cuda()
    zero = torch.zeros(H, H, device="cuda")
    mu, sigma = r(H, H), r(H, H) + 3
    smu, ssig, sw = r(D, H), 3 + 5 * r(D, H), r(D, H)
    serev = torch.where(r(D, H) < 0.5, 1.0, -1.0)
    cm, gl, vl = 2 + r(H), r(H), r(H) - 0.5
    out, last = ltc_cuda.ltc_cuda_forward(x, h0, zero, zero, mu, sigma, smu, ssig, serev, sw, cm, gl, vl, 1, eps)
    num, den = ltc_cuda._cuda_module.ltc_sensory_fwd(x.reshape(B * T, D), ssig, smu, sw, serev)
    total = (cm + gl + den + eps).reshape(B, T, H)
    h, hl = ltc_cuda.ltc_linear_scan(cm / total, (gl * vl + num).reshape(B, T, H) / total, h0)
    # tanh.approx gates and the sensory sums are shared; what differs are fp32 roundings
    assert torch.allclose(out, h, rtol=0, atol=1e-4) and torch.allclose(last, hl, rtol=0, atol=1e-4)
