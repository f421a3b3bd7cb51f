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
