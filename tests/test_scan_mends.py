"""GPU: calls of the scans that were once answered wrongly, refused, or by luck."""
import ctypes

import pytest
import torch

import ltc_cuda
from sequence_ref import assert_within, scan_reference

pytestmark = pytest.mark.gpu


def operands(op, lead, H, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    if op == "linear":
        args = {"a": torch.rand(*lead, H, generator=g) * 1.2 - 0.2, "b": r(*lead, H)}
    else:
        args = {"x": r(*lead, H), "rate": r(*lead, H).clamp(-4, 4), "gate": r(*lead, H).clamp(-4, 4)}
    args = {n: t.to(dtype).cuda() for n, t in args.items()}
    if op == "gated":
        args["decay"] = (r(H) - 3).cuda()
    return args


def run(op, args, h0=None, starts=None):
    fn = ltc_cuda.ltc_linear_scan if op == "linear" else ltc_cuda.ltc_gated_scan
    return fn(*args.values(), h0, seq_starts=starts)


def cluster_of(B, T, H, S=0):
    p = ltc_cuda.LtcScanPlan()
    assert ltc_cuda._lib.ltc_scan_plan(ctypes.byref(ltc_cuda.LtcScanDims(B, T, H, 0, S)), ctypes.byref(p)) == 0
    return p.cluster


@pytest.mark.parametrize("op", ["linear", "gated"])
@pytest.mark.parametrize("T,H,cluster", [(1100, 20, 8), (2100, 1100, 4), (9000, 9, 16)])
def test_clusters_close_together(op, T, H, cluster):
    """Blocks of a cluster leave behind one barrier, the ones without a channel or an end to write
    too; no wait expires."""
    assert cluster_of(1, T, H) >= cluster
    args = operands(op, (1, T), H, T)
    ref = scan_reference(op, args, None)
    for starts in (None, torch.tensor([0, 3, 3, T // 2, T - 5], device="cuda")):
        leaves = {n: t.clone().requires_grad_(True) for n, t in args.items()}
        call = leaves if starts is None else {n: t if n == "decay" else t[0] for n, t in leaves.items()}
        h, last = run(op, call, None, starts)
        (h.sum() + last.sum()).backward()
        if starts is None:
            assert_within(h, *ref["h"], "h")
        assert all(torch.isfinite(t.grad).all() for t in leaves.values())
    assert ltc_cuda.wait_timeouts() == 0


def test_wide_rows_of_one_time_step():
    """One position of a projection whose rows are more than 2^28 elements apart: a step, and a scan of T = 1."""
    H, apart = 8, (1 << 28) + 16
    store = torch.zeros(apart + 3 * H, device="cuda", dtype=torch.float16)
    g = torch.Generator().manual_seed(0)
    rows = torch.randn(2, 3 * H, generator=g).half().cuda()
    store[:3 * H], store[apart:] = rows[0], rows[1]
    wide = store.as_strided((2, 3 * H), (apart, 1))
    decay, state = torch.randn(H, generator=g).cuda() - 3, torch.randn(2, H, generator=g).cuda()
    want = ltc_cuda.ltc_gated_scan_step(*rows.split(H, dim=1), decay, state)
    got = ltc_cuda.ltc_gated_scan_step(*wide.split(H, dim=1), decay, state)
    assert all(torch.equal(u, v) for u, v in zip(got, want))
    leaf = rows[:, None].clone().requires_grad_(True)  # T = 1, with a time stride that means nothing
    far = [t.as_strided((2, 1, H), (apart, apart, 1), t.storage_offset()) for t in wide.split(H, dim=1)]
    for t in far:
        t.requires_grad_(True)
    h, last = ltc_cuda.ltc_gated_scan(*far, decay, state)
    hw, lw = ltc_cuda.ltc_gated_scan(*leaf.split(H, dim=2), decay, state)
    assert torch.equal(h, hw) and torch.equal(last, lw) and torch.equal(last, want[1])
    grads = torch.autograd.grad([h, last], far, [torch.ones_like(h), torch.ones_like(last)])
    (gw,) = torch.autograd.grad([hw, lw], [leaf], [torch.ones_like(h), torch.ones_like(last)])
    assert torch.equal(torch.cat(grads, 2), gw)


def gradients(op, args, h0, dh, dlast, starts):
    leaves = {n: t.clone().requires_grad_(True) for n, t in args.items()}
    first = h0.clone().requires_grad_(True)
    h, last = run(op, leaves, first, starts)
    grads = torch.autograd.grad([h, last], [*leaves.values(), first], [dh, dlast])
    return {"h": h, "state": last, **{"d" + n: g for n, g in zip([*leaves, "h0"], grads)}}


def dirty_memory(*like):
    """What the allocator hands out next has been written before."""
    held = [torch.full_like(t, 1e30) for t in like for _ in range(8)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("op", ["linear", "gated"])
@pytest.mark.parametrize("H", [12, 5])
@pytest.mark.parametrize("starts,N,wide", [
    ([0, 40, 90], 70, False), ([-5, 30, 200, 300], 130, False), ([0, 700, 5000, 6000], 1500, False),
    ([0, 64, 128, 129], 128, False), ([0, 30, (1 << 32) + 7, 1 << 40], 90, True)])
def test_offsets_end_at_the_tokens(op, starts, N, wide, H):
    """A sequence that reaches past the tokens ends with them, one behind them has none; int64
    offsets do not wrap.  Both kinds of state rows are written."""
    S = len(starts) - 1
    args = operands(op, (N,), H, N + H)
    g = torch.Generator().manual_seed(N)
    h0, dh, dlast = (torch.randn(*s, generator=g).cuda() for s in ((S, H), (N, H), (S, H)))
    t = torch.tensor(starts, device="cuda", dtype=torch.int64 if wide else torch.int32)
    dirty_memory(h0, dh)
    got = gradients(op, args, h0, dh, dlast, t)
    ref = scan_reference(op, args, h0, dh, dlast, [min(max(s, 0), N) for s in starts])
    for n, v in got.items():
        assert_within(v, *ref[n], n)


@pytest.mark.parametrize("op", ["linear", "gated"])
@pytest.mark.parametrize("starts,N", [([0, 100, 50, 60], 200), ([90, 3, 500, -7, 20], 400), ([10, 5], 40),
                                      ([0, 1500, 300, 2000], 2000)])
def test_offsets_out_of_order_give_nan_states(op, starts, N):
    """Never what was in memory before: states and their gradients are NaN, all of them."""
    S, H = len(starts) - 1, 20
    args = operands(op, (N,), H, N)
    h0 = torch.zeros(S, H, device="cuda")
    t = torch.tensor(starts, device="cuda", dtype=torch.int32)
    dirty_memory(h0)
    got = gradients(op, args, h0, torch.ones(N, H, device="cuda"), torch.ones(S, H, device="cuda"), t)
    assert got["state"].isnan().all() and got["dh0"].isnan().all()


def many_sequences(kind, N):
    g = torch.Generator().manual_seed(7)
    if kind == "short":  # about 1600 sequences of 0 to 3 tokens: lanes search more than 32 offsets each
        lens = torch.randint(0, 4, (1600,), generator=g)
        starts = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)])
        return [int(s) for s in starts if s <= N]
    if kind == "runs of empty ones":  # inside tiles, between their threads, at both ends
        at = torch.tensor([0, 5, 37, 63, 64, 130, 131, N - 1, N]).repeat_interleave(400)
        return at.tolist()
    return [0, 3] + [70] * 20000 + [100, 100, N]  # one offset, inside a tile


@pytest.mark.parametrize("op", ["linear", "gated"])
@pytest.mark.parametrize("N,H", [(700, 5), (2300, 12)])
@pytest.mark.parametrize("kind", ["short", "runs of empty ones", "one offset"])
def test_more_than_1024_sequences(op, N, H, kind):
    starts = many_sequences(kind, N)
    S = len(starts) - 1
    args = operands(op, (N,), H, S)
    g = torch.Generator().manual_seed(S)
    h0, dh, dlast = (torch.randn(*s, generator=g).cuda() for s in ((S, H), (N, H), (S, H)))
    got = gradients(op, args, h0, dh, dlast, torch.tensor(starts, device="cuda", dtype=torch.int32))
    ref = scan_reference(op, args, h0, dh, dlast, starts)
    for n, v in got.items():
        assert_within(v, *ref[n], n)


def test_many_empty_sequences_are_stepped_over():
    """A million empty sequences at one offset inside a tile, while the cluster's other blocks wait
    for it: no bounded wait expires, and the tokens are those of the two sequences around them."""
    N, H, S = 2000, 16, 1000002
    assert cluster_of(1, N, H, S) > 1
    args = operands("gated", (N,), H, 3)
    starts = torch.full((S + 1,), 1030, dtype=torch.int32, device="cuda")
    starts[0], starts[-1] = 0, N
    h, last = run("gated", args, None, starts)
    want, wl = run("gated", args, None, torch.tensor([0, 1030, N], dtype=torch.int32, device="cuda"))
    assert torch.equal(h, want) and torch.equal(last[[0, -1]], wl) and bool((last[1:-1] == 0).all())
    assert ltc_cuda.wait_timeouts() == 0


def test_step_output_overlapping_an_operand_is_refused():
    """The checks that the binding makes first agree with the ones behind them."""
    z, d, pool = torch.zeros(2, 4, device="cuda"), torch.zeros(4, device="cuda"), torch.zeros(64, device="cuda")
    out = pool[8:16].view(2, 4)
    for args in ((pool[10:18].view(2, 4), z, z, d, z), (z, z, pool[6:30].view(2, 12)[:, :4], d, z),
                 (z, z, z, pool[8:12], z), (z, z, z, d, pool[9:17].view(2, 4))):
        with pytest.raises(ValueError, match="overlap"):
            ltc_cuda.ltc_gated_scan_step(*args, out_state=out)
    pool.copy_(torch.randn(64, generator=torch.Generator().manual_seed(0)))
    x = out.clone()
    want = ltc_cuda.ltc_gated_scan_step(x, x, x, d, x)[1]
    assert ltc_cuda.ltc_gated_scan_step(out, out, out, d, out, out_state=out)[1] is out and torch.equal(out, want)
