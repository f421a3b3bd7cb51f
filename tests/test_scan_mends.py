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
