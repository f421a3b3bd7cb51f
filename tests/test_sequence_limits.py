"""CPU: the sequence operators' limits, at the value that is still taken and the first that is not."""
import ctypes

import pytest
import torch

import ltc_cuda


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_packed_sequences_past_2_30_are_refused(monkeypatch):
    """The search among the offsets adds two sequence indices: past 2^30 the sum wraps to an offset
    in front of the array."""
    args = t(4, 3), t(4, 3)
    for n in ((1 << 30) + 1, (1 << 31) - 1):
        starts = t(1, dtype=torch.int32).expand(n + 1)
        with pytest.raises(ValueError, match="sequences"):
            ltc_cuda.ltc_linear_scan(*args, seq_starts=starts)
    with pytest.raises(ValueError, match="the sm_100a kernels need CUDA"):  # taken, up to the device
        ltc_cuda.ltc_linear_scan(*args, seq_starts=t(1, dtype=torch.int32).expand((1 << 30) + 1))
    lib = ltc_cuda._lib
    if lib is None:
        pytest.skip("library not built")
    dims = ltc_cuda.LtcScanDims(1, 4, 3, 0, (1 << 30) + 1)
    assert lib.ltc_scan_plan(ctypes.byref(dims), ctypes.byref(ltc_cuda.LtcScanPlan())) != 0
    assert b"packed sequences" in lib.ltc_last_error()
    # one fewer gets as far as the device
    dims.num_seqs -= 1
    lib.ltc_scan_plan(ctypes.byref(dims), ctypes.byref(ltc_cuda.LtcScanPlan()))
    assert b"packed sequences" not in lib.ltc_last_error()


def test_time_stride_of_a_single_step_is_not_looked_at(monkeypatch):
    """Past 2^28 elements a time stride is refused, but one step has no use for any."""
    monkeypatch.setattr(ltc_cuda, "_on_cuda", lambda *_: None)
    one = t(1).as_strided((1, 1, 1), (1, (1 << 28) + 1, 1))
    (a, _), _, _, dims = ltc_cuda._scan_operands(("a", "b"), (one, one), None, None)
    assert a.stride(1) > 1 << 28 and dims == (1, 1, 1, 0)
    two = torch.empty(1).as_strided((1, 1, 1), (1, 1, 1)).expand(1, 2, 1)
    ltc_cuda._scan_operands(("a", "b"), (two, two), None, None)
    wide = torch.empty(((1 << 28) + 2,), dtype=torch.float16).as_strided((1, 2, 1), (1, (1 << 28) + 1, 1))
    with pytest.raises(ValueError, match="time stride"):
        ltc_cuda._scan_operands(("a", "b"), (wide, wide), None, None)


def test_scale_has_to_fit_fp32(monkeypatch):
    """Positive and finite as a double is not enough: 1e39 is infinite and 1e-50 is 0 to the kernels."""
    monkeypatch.setattr(ltc_cuda, "_on_cuda", lambda *_: None)
    for scale in (1e39, 1e-50, 0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            ltc_cuda.ltc_gated_scan(t(1, 2, 3), t(1, 2, 3), t(1, 2, 3), t(3), scale=scale)
        with pytest.raises(ValueError, match="scale"):
            ltc_cuda.ltc_gated_scan_step(t(2, 3), t(2, 3), t(2, 3), t(3), t(2, 3), scale=scale)
    for scale in (8, 8.0, torch.tensor(8.0), 3e38):
        ltc_cuda._check_decay(t(3), t(3).device, 3, scale)
    lib = ltc_cuda._lib
    if lib is None:
        pytest.skip("library not built")
    dims = ctypes.byref(ltc_cuda.LtcScanDims(1, 2, 3, 0, 0))
    for scale in (float("inf"), float("nan"), 0.0, -2.0):
        for rc in (lib.ltc_gated_scan_step(dims, None, None, None, None, scale, None, None, None, None),
                   lib.ltc_gated_scan_forward(dims, None, None, None, None, scale, *[None] * 6, 0, None),
                   lib.ltc_gated_scan_backward(dims, None, None, None, None, scale, *[None] * 11, 0, None)):
            assert rc != 0 and b"scale" in lib.ltc_last_error()


def test_step_output_may_not_overlap_an_operand(monkeypatch):
    """Threads of other rows would read what one has written already.  The same array is no
    overlap: each element is read and written by one thread."""
    monkeypatch.setattr(ltc_cuda, "_on_cuda", lambda *_: None)
    monkeypatch.setattr(ltc_cuda, "_torch_binding", None)
    z, d, pool = t(2, 4), t(4), t(64)
    out = pool[8:16].view(2, 4)
    for args in ((pool[10:18].view(2, 4), z, z, d, z), (z, pool[4:12].view(2, 4), z, d, z),
                 (z, z, pool[6:30].view(2, 12)[:, :4], d, z), (z, z, z, pool[8:12], z), (z, z, z, pool[13:17], z),
                 (z, z, z, d, pool[9:17].view(2, 4))):
        with pytest.raises(ValueError, match="overlap"):
            ltc_cuda.ltc_gated_scan_step(*args, out_state=out)
    joint = t(3, 24)
    for args, to in (((out, z, z, d, z), out), ((z, z, z, d, out), out), ((z, out, out, d, out), out),
                     ((z, z, z, pool[:4], pool[16:24].view(2, 4)), out),
                     ((*joint[:2, :12].split(4, dim=1), d, z), joint.view(-1)[48:56].view(2, 4)),
                     ((out.t().contiguous().t(), z, z, d, z), out)):
        with pytest.raises(RuntimeError):  # taken, as far as the kernels
            ltc_cuda.ltc_gated_scan_step(*args, out_state=to)
