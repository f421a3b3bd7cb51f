"""CPU: data_parallel by itself, as a program uses it whose model is not from this package."""
import os
import subprocess
import sys

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

_CHILD = r'''
import importlib.util, sys, torch
spec = importlib.util.spec_from_file_location("data_parallel", sys.argv[1])
dp = importlib.util.module_from_spec(spec)
spec.loader.exec_module(dp)

class Model(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.w = torch.nn.Parameter(torch.ones(3, 2))
    def forward(self, x):
        return x @ self.w, None

m = Model()
bucket = dp.FlatGradBucket(m.parameters())
dp.training_step(m, torch.ones(4, 3), bucket, torch.optim.SGD(m.parameters(), lr=0.5))
assert torch.equal(m.w.detach(), torch.full((3, 2), -1.0)) and dp.shard_range(5, 1, 2) == (3, 5)
assert "ltc_cuda" not in sys.modules
print("ALONE_OK")
'''


def test_the_plain_step_does_not_load_the_kernels():
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    path = os.path.join(REPO, "ltc-cuda_b200", "data_parallel.py")
    r = subprocess.run([sys.executable, "-c", _CHILD, path], capture_output=True, text=True, timeout=300, env=env,
                       cwd=os.path.dirname(REPO))
    assert r.returncode == 0 and "ALONE_OK" in r.stdout, r.stderr[-2000:]
