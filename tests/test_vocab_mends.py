"""GPU: calls of the vocabulary operators that were once answered wrongly, or by luck."""
import pytest
import torch

import ltc_cuda

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = float("inf")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows", [40, 4000])  # blocks of 256 and of 128 threads
@pytest.mark.parametrize("V,left", [(40, 40), (300, 300), (1500, 1500), (9000, 30)])
def test_alternatives_where_warps_hold_no_values(rows, V, left, dtype):
    """Short rows and rows whose mask leaves little take their threshold from all threads' maxima,
    behind a barrier that every warp has to meet: ids and their number, row by row."""
    g = torch.Generator().manual_seed(V + rows)
    z = (torch.randn(rows, V, generator=g) * 3).to(dtype).cuda()
    if left < V:
        keep = torch.rand(rows, V, generator=g).cuda().topk(left, dim=1).indices
        z = torch.full_like(z, -INF).scatter_(1, keep, z.gather(1, keep))
    z[1::7] = -INF
    tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
    order = torch.sort(z.float(), dim=1, descending=True, stable=True)
    for k in (1, 20, 33):
        want = torch.where(order.values[:, :k] > -INF, order.indices[:, :k], -1)
        for _ in range(5):
            assert torch.equal(ltc_cuda.ltc_token_logprobs(z, tokens, top_k=k).top_ids, want)
