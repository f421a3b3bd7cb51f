"""GPU: the sequence operators in the checked build (index checks counted instead of faulting):
packed sequences, also with offsets out of order, and the top entries, report no failed check."""
import os
import subprocess
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(REPO, "ltc-cuda_b200")
CHECKED = os.path.join(PKG, "libltc_sm100_checked.so")

_CHILD = r'''
import ctypes, torch
import ltc_cuda
lib = ctypes.CDLL(ltc_cuda.LIB_PATH)
assert lib.ltc_checked_build() > 0, "not the checked build"
g = torch.Generator().manual_seed(0)
r = lambda *s: torch.randn(*s, generator=g).cuda()
for H in (8, 13, 700):
    for starts in ([0, 3, 3, 90, 400], [0, 0, 0, 400, 400], [5, 300], [90, 3, 500, -7, 20], [400, 0], list(range(0, 401, 2))):
        leaves = [r(400, H).requires_grad_(True) for _ in range(3)] + [(r(H) - 3).requires_grad_(True)]
        h0 = r(len(starts) - 1, H).requires_grad_(True)
        h, last = ltc_cuda.ltc_gated_scan(*leaves, h0, seq_starts=torch.tensor(starts, device="cuda"))
        torch.autograd.grad(h.sum() + last.nan_to_num().sum(), leaves + [h0])
for V in (5, 129, 3001, 70001):
    for dt in (torch.float32, torch.bfloat16):
        z = r(3, V).to(dt)
        z[1] = 0
        ltc_cuda.ltc_token_logprobs(z, torch.zeros(3, dtype=torch.int64, device="cuda"), top_k=min(V, 64))
        ltc_cuda.ltc_token_logprobs(z.repeat(500, 1), torch.zeros(1500, dtype=torch.int64, device="cuda"), top_k=3)
count, site = ctypes.c_int(-1), ctypes.c_int(-1)
assert lib.ltc_check_errors(ctypes.byref(count), ctypes.byref(site)) == 0
assert count.value == 0, f"{count.value} failed index checks, first at site {site.value}"
assert ltc_cuda.wait_timeouts() == 0
print("SEQUENCE_CHECKED_OK")
'''


@pytest.mark.gpu
@pytest.mark.skipif(not os.path.exists(CHECKED), reason="checked build not built (ltc-cuda_b200/build.py --checked)")
def test_checked_build_of_the_sequence_operators():
    env = dict(os.environ, LTC_SM100_LIB=CHECKED)
    env["PYTHONPATH"] = os.pathsep.join([PKG, REPO] + [p for p in env.get("PYTHONPATH", "").split(os.pathsep) if p])
    r = subprocess.run([sys.executable, "-c", _CHILD], capture_output=True, text=True, timeout=600, env=env, cwd=REPO)
    assert r.returncode == 0 and "SEQUENCE_CHECKED_OK" in r.stdout, (r.stdout + r.stderr)[-3000:]
