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


@pytest.mark.parametrize("V", [33, 5000])
@pytest.mark.parametrize("exponent", [0, -30, -60])
def test_entropy_gradient_of_masked_rows_under_large_factors(V, exponent):
    """A loss scale of 2^40 over temperatures down to 2^-60: powers of two, so every value is that
    of the plain call times the factor, bit by bit, and masked entries get 0."""
    g = torch.Generator().manual_seed(V)
    z = torch.randn(4, V, generator=g).cuda() * 3
    z[0, ::3] = -INF
    z[1, 1:] = -INF
    z[2, ::5] = -1e4
    z[3] = -INF
    tokens = torch.zeros(4, dtype=torch.int64, device="cuda")
    tau, factor = 2.0 ** exponent, 2.0 ** 40

    def grad(logits, temperature, scale):
        leaf = logits.clone().requires_grad_(True)
        r = ltc_cuda.ltc_token_logprobs(leaf, tokens, temperature=temperature)
        w = torch.full((4,), scale, device="cuda")
        return torch.autograd.grad([r.logprobs, r.entropy], [leaf], [w, w])[0]

    want = grad(z, 1.0, 1.0)
    # the gradient at the token is its own weight less q's share, at a masked token too
    masked = z.isneginf() & (torch.arange(V, device="cuda") > 0)
    assert torch.isfinite(want).all() and bool((want[masked] == 0).all()) and bool((want[0, 1::3] != 0).any())
    got = grad(z * tau, tau, factor)
    expected = (want.double() * factor / tau).float()
    # what the plain call holds below 2^-80 may have been rounded as a subnormal number
    sure = (want.abs() > 2.0 ** -80) | (want == 0)
    finite = torch.isfinite(expected) & sure
    assert torch.equal(got[finite], expected[finite])
    assert not got.isnan().any() and bool((got[masked] == 0).all())


@pytest.mark.parametrize("exponent,near", [(-60, False), (-80, False), (40, True), (70, True)])
def test_distillation_at_extreme_temperatures(exponent, near):
    """tau^2 by itself is 0 or infinite there, the loss is not.  Powers of two: the loss is that of
    temperature 1 times tau^2, bit by bit, and a row without entries costs 0."""
    g = torch.Generator().manual_seed(1)
    z = torch.randn(5, 2, generator=g).cuda()
    ids = torch.tensor([[0, 1]] * 4 + [[-1, -1]], device="cuda")
    if near:  # a loss of about 2^-19 .. 2^-15
        teacher = z + torch.tensor([0.0, 2.0 ** -6], device="cuda")
    else:     # a loss of about 2^40
        z[:, 1] -= 2.0 ** 40
        teacher = torch.tensor([-(2.0 ** 40), 0.0], device="cuda").expand(5, 2).contiguous()
    tau = 2.0 ** exponent
    plain = ltc_cuda.ltc_distill_loss(z, ids, teacher)
    assert plain[4] == 0 and bool((plain[:4] > 0).all()) and bool(torch.isfinite(plain).all())
    expected = (plain.double() * tau * tau).float()
    assert bool((expected[:4] > 2.0 ** -126).all()) and bool(torch.isfinite(expected).all())
    assert torch.equal(ltc_cuda.ltc_distill_loss(z * tau, ids, teacher * tau, temperature=tau), expected)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_zero_gradients_of_rows_with_an_id_past_the_vocabulary(dtype):
    """A row that a zero weight takes out of the loss gets zeros, also where its id makes its loss NaN."""
    z = torch.randn(3, 300, generator=torch.Generator().manual_seed(0)).to(dtype).cuda()
    ids = torch.tensor([[1, 300], [2, 3], [1 << 40, -1]], device="cuda")
    leaf = z.clone().requires_grad_(True)
    w = torch.tensor([0.0, 1.0, 2.0], device="cuda")
    loss = ltc_cuda.ltc_distill_loss(leaf, ids, torch.zeros(3, 2, device="cuda"))
    (g,) = torch.autograd.grad([loss], [leaf], [w])
    assert (g[0] == 0).all() and torch.isfinite(g[1]).all() and g[2].isnan().any() and (g[1] != 0).any()
    r = ltc_cuda.ltc_token_logprobs(leaf, ids[:, 1])
    assert r.logprobs.isnan().tolist() == [True, False, False]
    (g,) = torch.autograd.grad([r.logprobs], [leaf], [w])
    assert (g[0] == 0).all() and (g[1] != 0).any() and (g[2] == 0).all()
    (g,) = torch.autograd.grad([ltc_cuda.ltc_token_logprobs(leaf, ids[:, 1]).logprobs], [leaf], [w + 1])
    assert g[0].isnan().any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("tau", [0.25, 1.0, 2.0])
def test_distillation_of_entries_masked_by_the_lowest_value(dtype, tau):
    """A teacher's entry that the student masks with the type's lowest value costs p |lowest| tau:
    a loss within fp32's range, where |lowest| / (tau ln 2) is not."""
    g = torch.Generator().manual_seed(3)
    z = torch.randn(6, 700, generator=g).to(dtype).cuda()
    ids = torch.randint(0, 700, (6, 5), generator=g).cuda()
    teacher = torch.randn(6, 5, generator=g).cuda() * 2
    teacher[:, 0] -= 8
    low = torch.finfo(dtype).min
    z[torch.arange(6, device="cuda"), ids[:, 0]] = low
    loss = ltc_cuda.ltc_distill_loss(z, ids, teacher, temperature=tau)
    w, t = z.cpu().double() / tau, teacher.cpu().double() / tau
    p = torch.softmax(t, 1)
    want = tau * tau * (p * (torch.log_softmax(t, 1) - torch.log_softmax(w, 1).gather(1, ids.cpu()))).sum(1)
    assert bool((want < 3e38).all()) and bool((want > 1e12).all())  # all but nothing is the masked entry's
    # p of that entry is off by 4 U times its distance from the largest and 25 U more (two exponentials, the sum
    # of five, a division); the products and the sum round ten times
    off = (4 * (t.max(1).values - t[:, 0]) + 35) * 2.0 ** -24
    assert bool(((loss.cpu().double() - want).abs() <= off * want).all())
