"""GPU: ltc_distill_loss and ltc_token_logprobs against their fp64 definitions."""
import pytest
import torch

import ltc_cuda
from sequence_ref import U, assert_within, half_step, vocab_reference

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = float("inf")


def logits_of(rows, V, dtype, seed, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, V, generator=g) * scale).to(dtype).cuda()


def grad_bound(ref, alpha, beta, alpha_err, extra, dz, dtype):
    """q (alpha + beta log q) + extra: q is off by tol_log and 3 ulp, log q by tol_log, alpha by
    alpha_err and 3 ulp; the sum is rounded twice and then once to the output's type."""
    lq = torch.where(ref["q"] > 0, ref["logq"].abs(), 0.0)
    qerr = ref["q"] * (ref["tol_log"] + 6 * U)
    return (qerr * (alpha.abs() + beta.abs() * lq) + ref["q"] * (beta.abs() * (ref["tol_log"] + 3 * U * lq)
            + alpha_err + 6 * U * alpha.abs()) + 4 * U * extra.abs() + (half_step(dtype) + 2 * U) * dz.abs()
            + torch.finfo(dtype).tiny * torch.finfo(dtype).eps)


def check_scores(z, tokens, tau=1.0, k=0, grads=True, dtype=None):
    dtype = z.dtype
    rows, V = z.shape
    leaf = z.detach().requires_grad_(grads)
    r = ltc_cuda.ltc_token_logprobs(leaf, tokens, top_k=k, temperature=tau)
    ref = vocab_reference("scores", z, tau)
    tok = tokens.cpu().long()
    given = tok >= 0
    at = tok.clamp(min=0)[:, None]
    lp = torch.where(given, ref["logq"].gather(1, at)[:, 0], 0.0)
    tol = torch.where(given, ref["tol_log"].gather(1, at)[:, 0], 0.0)
    assert_within(r.logprobs, lp, tol, "logprobs")
    assert_within(r.entropy, ref["ent"], ref["tol_ent"], "entropy")
    if k:
        order = torch.sort(z.cpu().float(), dim=1, descending=True, stable=True)
        ids = torch.where(order.values[:, :k] > -INF, order.indices[:, :k], -1)
        assert torch.equal(r.top_ids.cpu(), ids)
        best = order.indices[:, :k]
        assert_within(r.top_logprobs, ref["logq"].gather(1, best), ref["tol_log"].gather(1, best), "top_logprobs")
    else:
        assert r.top_ids is None and r.top_logprobs is None
    if not grads:
        return r
    g = torch.Generator().manual_seed(5)
    glp, gent = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    (dz,) = torch.autograd.grad([r.logprobs, r.entropy], [leaf], [glp.cuda(), gent.cuda()])
    glp, gent = glp.double(), gent.double()
    hot = torch.zeros_like(ref["q"]).scatter_(1, at, given.double()[:, None])
    alpha = -(torch.where(given, glp, 0.0) + gent * ref["ent"])[:, None] / tau
    beta = -gent[:, None] / tau
    extra = hot * glp[:, None] / tau
    want = ref["q"] * alpha + beta * ref["flat"] + extra
    want = torch.where(ref["live"], want, 0.0)
    assert dz.dtype == dtype
    bound = grad_bound(ref, alpha, beta, (gent.abs() * ref["tol_ent"])[:, None] / tau, extra, want, dtype)
    assert_within(dz, want, bound, "dlogits")
    return r


SHAPES = [(1, 1), (3, 2), (5, 7), (4, 31), (2, 1000), (3, 1793), (9, 4099), (2, 8192), (3, 20001), (1, 40000)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,V", SHAPES)
@pytest.mark.parametrize("tau", [1.0, 0.6])
def test_scores(rows, V, dtype, tau):
    z = logits_of(rows, V, dtype, rows + V)
    tokens = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(V)).cuda()
    if rows > 2:
        tokens[1] = -1
    check_scores(z, tokens, tau, k=min(V, 5))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("k", [1, 8, 9, 33, 64])
@pytest.mark.parametrize("V", [64, 3001, 70000])
def test_top_counts(k, V, dtype):
    z = logits_of(3, V, dtype, k * V)
    check_scores(z, torch.zeros(3, dtype=torch.int32, device="cuda"), k=k, grads=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two values", "late", "early", "sparse", "one lane"])
@pytest.mark.parametrize("V", [100, 9000, 33001])
def test_top_of_awkward_rows(kind, V, dtype):
    """Ties everywhere, sorted rows (the list overruns and the row is searched), masked
    halves, and large values that all fall to one thread."""
    z = logits_of(2, V, dtype, V)
    if kind == "equal":
        z.fill_(0.25)
    elif kind == "rising":
        z = z.float().sort(dim=1).values.to(dtype)
    elif kind == "falling":
        z = z.float().sort(dim=1, descending=True).values.to(dtype)
    elif kind == "two values":
        z = torch.where(z > 0, 1.0, -1.0).to(dtype)
    elif kind == "late":
        z[:, :-7] = -INF
    elif kind == "early":
        z[:, 7:] = -INF
    elif kind == "sparse":
        keep = torch.zeros(V, dtype=torch.bool, device="cuda")
        keep[torch.randperm(V, generator=torch.Generator().manual_seed(1))[:12].cuda()] = True
        z.masked_fill_(~keep, -INF)
    else:
        z[:, ::2048] += 20
    check_scores(z, torch.tensor([0, V - 1], device="cuda"), k=20, grads=kind != "rising")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_masks_and_lowest_values(dtype):
    """-inf entries, the type's lowest value as a mask (also alone in its row, also under a
    small temperature), rows whose mask leaves nothing or one entry."""
    low = torch.finfo(dtype).min
    z = logits_of(7, 3000, dtype, 1)
    z[0, ::3] = -INF
    z[1, ::3] = low
    z[2] = low
    z[3] = -INF
    z[4] = -INF
    z[4, 77] = 1.5
    z[5] = low
    z[5, 2999] = 3.0
    z[6] = torch.finfo(dtype).max
    tokens = torch.tensor([0, 3, 5, 6, 77, 2999, 9], device="cuda")
    for tau in (1.0, 0.25):
        r = check_scores(z, tokens, tau, k=6)
    assert r.logprobs[0] == -INF and r.logprobs[3] == -INF and r.entropy[3] == 0
    assert r.top_ids[3].tolist() == [-1] * 6 and r.top_ids[4].tolist() == [77] + [-1] * 5
    assert abs(r.entropy[2].item() - torch.log(torch.tensor(3000.0)).item()) < 1e-4


def test_nan_and_infinite_logits_make_their_rows_nan():
    z = logits_of(4, 5000, torch.float32, 3)
    z[0, 17] = float("nan")
    z[1, 4999] = INF
    z[2] = -INF
    z[2, 5] = float("nan")
    leaf = z.clone().requires_grad_(True)
    r = ltc_cuda.ltc_token_logprobs(leaf, torch.tensor([3, 3, 3, 3], device="cuda"), top_k=3)
    assert r.logprobs.isnan().tolist() == [True, True, True, False]
    assert r.entropy.isnan().tolist() == [True, True, True, False]
    (g,) = torch.autograd.grad(r.logprobs.sum(), leaf)
    assert g[:3].isnan().any(dim=1).all() and torch.isfinite(g[3]).all()
    loss = ltc_cuda.ltc_distill_loss(z, torch.full((4, 1), 3, device="cuda"), torch.zeros(4, 1, device="cuda"))
    assert loss.isnan().tolist() == [True, True, True, False]


def check_distill(z, ids, teacher, tau=1.0):
    rows, V = z.shape
    leaf = z.detach().requires_grad_(True)
    loss = ltc_cuda.ltc_distill_loss(leaf, ids, teacher, temperature=tau)
    g = torch.rand(rows, generator=torch.Generator().manual_seed(2)) + 0.5
    (dz,) = torch.autograd.grad([loss], [leaf], [g.cuda()])
    ref = vocab_reference("distill", z, tau)
    idc, t = ids.cpu().long(), teacher.detach().cpu().double() / tau
    there = (idc >= 0) & (t > -INF)
    any_ = there.any(1, keepdim=True)
    p = torch.softmax(torch.where(there, t, -INF).masked_fill(~any_, 0.0), dim=1) * there
    logp = torch.where(p > 0, p.log(), 0.0)
    at = idc.clamp(min=0)
    lq = torch.where(p > 0, ref["logq"].gather(1, at), 0.0)
    want = tau * tau * (p * (logp - lq)).sum(1)
    # p is a softmax of K <= 256 entries like q: off by perr; log q by tol_log
    span = torch.where(there, (t - torch.where(there, t, -INF).max(1, keepdim=True).values).abs(), 0.0)
    perr = 4 * U * span + (20 + 3 * span.mean(1, keepdim=True)) * U + 3 * U * logp.abs()
    tol = (p * (perr * (1 + (logp - lq).abs()) + ref["tol_log"].gather(1, at) + 3 * U * (logp.abs() + lq.abs()))
           + 12 * U * (p * (logp - lq)).abs()).sum(1) * tau * tau
    tol = torch.where(want.isinf(), 0.0, tol.nan_to_num())
    assert_within(loss, want, tol, "loss")
    gg = (g.double() * tau)[:, None]
    hot = torch.zeros_like(ref["q"]).scatter_add_(1, at, p)
    hot_err = torch.zeros_like(ref["q"]).scatter_add_(1, at, p * (perr + 8 * U))
    alpha = torch.where(any_, gg, 0.0)
    dwant = torch.where(ref["live"], alpha * ref["q"] - gg * hot, 0.0)
    bound = grad_bound(ref, alpha, torch.zeros_like(alpha), torch.zeros_like(alpha), gg * hot, dwant, z.dtype)
    assert_within(dz, dwant, bound + gg * hot_err, "dlogits")
    return loss, dz


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tdtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,K,tau", [(1, 1, 1, 1.0), (4, 33, 33, 2.0), (3, 1000, 5, 1.0), (7, 8193, 32, 0.5),
                                          (2, 20001, 256, 3.0), (1, 50000, 100, 1.0)])
def test_distill(rows, V, K, tau, dtype, tdtype):
    z = logits_of(rows, V, dtype, V + K)
    g = torch.Generator().manual_seed(K)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(rows)])
    teacher = (torch.randn(rows, K, generator=g) * 2).to(tdtype)
    if rows > 2:
        ids[0, K // 2:] = -1   # fewer entries
        ids[1] = -1            # none
        if K > 4:
            ids[2, 1::2] = ids[2, 0]           # the same id many times
            teacher[2, 3] = -INF               # a masked teacher entry
    loss, dz = check_distill(z, ids.cuda(), teacher.cuda(), tau)
    if rows > 2:
        assert (K == 1 or loss[1] == 0) and (dz[1] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_distill_masks(dtype):
    low = torch.finfo(dtype).min
    z = logits_of(6, 2000, dtype, 4)
    z[0, ::2] = -INF
    z[1] = -INF             # no student distribution
    z[2] = low
    z[3, 10] = -INF         # the teacher wants what the mask forbids: infinite loss
    ids = torch.tensor([[1, 3], [4, 5], [8, 9], [10, 11], [0, 1], [2, 3]], device="cuda")
    teacher = torch.randn(6, 2, generator=torch.Generator().manual_seed(1)).cuda()
    teacher[4] = -INF       # entries without any weight
    teacher[5] = torch.tensor([low, 0.0])
    loss, dz = check_distill(z, ids, teacher.to(dtype))
    assert loss[1] == INF and (dz[1] == 0).all() and loss[3] == INF and torch.isfinite(dz[3]).all()
    assert loss[4] == 0 and (dz[4] == 0).all()


def test_ids_past_the_vocabulary_are_loud():
    z = logits_of(3, 50, torch.float32, 8)
    leaf = z.clone().requires_grad_(True)
    loss = ltc_cuda.ltc_distill_loss(leaf, torch.tensor([[1, 50], [2, 3], [1 << 40, 0]], device="cuda"),
                                     torch.zeros(3, 2, device="cuda"))
    (g,) = torch.autograd.grad(loss.sum(), leaf)
    assert loss.isnan().tolist() == [True, False, True] and g.isnan().any(1).tolist() == [True, False, True]
    r = ltc_cuda.ltc_token_logprobs(leaf, torch.tensor([50, 3, 1 << 40], device="cuda"))
    (g,) = torch.autograd.grad(r.logprobs.sum(), leaf)
    assert r.logprobs.isnan().tolist() == [True, False, True] and torch.isfinite(r.entropy).all()
    assert g.isnan().any(1).tolist() == [True, False, True]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V", [64, 1001])
def test_strided_logits(V, dtype):
    """Slices of (B, T, V), padded rows, rows that start off 16 bytes, a broadcast row, V strided."""
    base = logits_of(4 * 9, V + 3, dtype, V).reshape(4, 9, V + 3)
    tokens = torch.randint(0, V, (4, 9), generator=torch.Generator().manual_seed(1)).cuda()
    views = {"shifted": (base[..., :V][:, :-1], tokens[:, 1:]), "padded": (base[..., 1:V + 1], tokens),
             "permuted": (base[..., :V].transpose(0, 1), tokens.T),
             "every other": (base[:, ::2, 2:V + 2], tokens[:, ::2]),
             "four dims": (base.reshape(2, 2, 9, V + 3)[:, :, 1:, :V], tokens.reshape(2, 2, 9)[:, :, 1:]),
             "one row": (base[0, 0, :V], tokens[0, 0]),
             "broadcast": (base[:1, :1, :V].expand(4, 9, V), tokens),
             "strided V": (base[..., :V].transpose(1, 2).contiguous().transpose(1, 2), tokens)}
    for name, (z, tok) in views.items():
        packed = z.contiguous().reshape(-1, V)
        leaf, flat = z.detach().requires_grad_(True), packed.detach().requires_grad_(True)
        r = ltc_cuda.ltc_token_logprobs(leaf, tok, top_k=3)
        f = ltc_cuda.ltc_token_logprobs(flat, tok.reshape(-1), top_k=3)
        assert r.logprobs.shape == tok.shape and r.top_ids.shape == (*tok.shape, 3), name
        assert torch.allclose(r.logprobs.reshape(-1), f.logprobs, rtol=1e-5, atol=1e-5), name
        assert torch.equal(r.top_ids.reshape(-1, 3), f.top_ids), name
        (g,) = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), leaf)
        (gf,) = torch.autograd.grad(f.logprobs.sum() + f.entropy.sum(), flat)
        assert g.shape == z.shape
        assert torch.allclose(g.reshape(-1, V).float(), gf.float(), rtol=4 * half_step(dtype), atol=1e-5), name
        ids = tok[..., None] if tok.dim() else tok[None]
        d = ltc_cuda.ltc_distill_loss(leaf, ids, torch.zeros(ids.shape, device="cuda"))
        assert torch.allclose(d, -r.logprobs, rtol=1e-5, atol=1e-5), name


def test_gradient_against_differences():
    """Central differences of the fp64 loss with step 1e-4 along a direction."""
    z = logits_of(3, 700, torch.float32, 2)
    ids = torch.randint(0, 700, (3, 9), generator=torch.Generator().manual_seed(3)).cuda()
    teacher = torch.randn(3, 9, generator=torch.Generator().manual_seed(4)).cuda()
    tok = ids[:, 0]
    leaf = z.clone().requires_grad_(True)
    r = ltc_cuda.ltc_token_logprobs(leaf, tok, temperature=0.8)
    total = ltc_cuda.ltc_distill_loss(leaf, ids, teacher, temperature=1.5).sum() + r.logprobs.sum() + 2 * r.entropy.sum()
    (g,) = torch.autograd.grad(total, leaf)

    def loss(w):
        lq = torch.log_softmax(w / 1.5, 1)
        p = torch.softmax(teacher.cpu().double() / 1.5, 1)
        s = 2.25 * (p * (p.log() - lq.gather(1, ids.cpu()))).sum()
        l2 = torch.log_softmax(w / 0.8, 1)
        return (s + l2.gather(1, tok.cpu()[:, None]).sum() - 2 * (l2.exp() * l2).sum()).item()

    for seed in range(3):
        d = torch.randn(3, 700, generator=torch.Generator().manual_seed(seed)).double()
        w = z.cpu().double()
        slope = (loss(w + 1e-4 * d) - loss(w - 1e-4 * d)) / 2e-4
        assert abs(slope - (g.cpu().double() * d).sum().item()) < 1e-5 * (g.cpu().double() * d).abs().sum().item() + 1e-6


def test_rows_without_a_gradient_are_not_read():
    """A zero gradient gives zeros even where the logits are NaN; one gradient may be absent."""
    z = logits_of(3, 4000, torch.bfloat16, 2)
    z[1] = float("nan")
    leaf = z.requires_grad_(True)
    r = ltc_cuda.ltc_token_logprobs(leaf, torch.tensor([1, -1, 2], device="cuda"))
    (g,) = torch.autograd.grad([r.logprobs], [leaf], [torch.tensor([1.0, 5.0, 0.0], device="cuda")])
    assert (g[1:] == 0).all() and (g[0] != 0).any()
    z2 = logits_of(3, 4000, torch.bfloat16, 6).requires_grad_(True)
    r = ltc_cuda.ltc_token_logprobs(z2, torch.tensor([1, 2, 2], device="cuda"))
    (ge,) = torch.autograd.grad([r.entropy], [z2], [torch.ones(3, device="cuda")])
    assert torch.isfinite(ge).all() and (ge != 0).any()


def test_deterministic_and_independent_of_the_batch():
    for rows, V in ((2, 40000), (700, 5003)):
        z = logits_of(rows, V, torch.bfloat16, 7)
        tok = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(1)).cuda()
        one = ltc_cuda.ltc_token_logprobs(z, tok, top_k=10)
        two = ltc_cuda.ltc_token_logprobs(z, tok, top_k=10)
        for u, v in zip(one, two):
            assert torch.equal(u, v)


def test_empty():
    z = torch.zeros(0, 5, device="cuda", requires_grad=True)
    r = ltc_cuda.ltc_token_logprobs(z, torch.zeros(0, dtype=torch.int64, device="cuda"), top_k=2)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 2)
    assert torch.autograd.grad(r.logprobs.sum(), z)[0].shape == (0, 5)
    loss = ltc_cuda.ltc_distill_loss(z, torch.zeros(0, 3, dtype=torch.int64, device="cuda"),
                                     torch.zeros(0, 3, device="cuda"))
    assert loss.shape == (0,)


def test_offsets_past_32_bits():
    """More than 2^31 logits: the last rows against the same rows alone, which are summed in another
    order (n = V / 128 + 16 additions: 530 U = 3e-5), so that a gradient may round the other way."""
    rows, V = 32800, 65536
    z = torch.empty(rows, V, device="cuda", dtype=torch.bfloat16).normal_(generator=torch.Generator("cuda").manual_seed(1))
    tok = torch.arange(rows, device="cuda") % V
    leaf = z.requires_grad_(True)
    r = ltc_cuda.ltc_token_logprobs(leaf, tok)
    (g,) = torch.autograd.grad(r.logprobs.sum(), leaf)
    tail = z.detach()[-600:].clone().requires_grad_(True)
    s = ltc_cuda.ltc_token_logprobs(tail, tok[-600:])
    (gt,) = torch.autograd.grad(s.logprobs.sum(), tail)
    assert torch.allclose(r.logprobs[-600:], s.logprobs, rtol=0, atol=6e-5)
    assert torch.allclose(r.entropy[-600:], s.entropy, rtol=0, atol=6e-4)
    assert torch.allclose(g[-600:].float(), gt.float(), rtol=2 * 2.0 ** -7, atol=0)


def test_streams_and_graphs():
    z, new = logits_of(5, 9000, torch.bfloat16, 1), logits_of(5, 9000, torch.bfloat16, 2)
    ids = torch.randint(0, 9000, (5, 7), generator=torch.Generator().manual_seed(1)).cuda()
    teacher = torch.randn(5, 7, generator=torch.Generator().manual_seed(2)).cuda()
    w = torch.rand(5, generator=torch.Generator().manual_seed(3)).cuda()

    def step(t):
        leaf = t.detach().requires_grad_(True)
        r = ltc_cuda.ltc_token_logprobs(leaf, ids[:, 0], top_k=4)
        loss = ltc_cuda.ltc_distill_loss(leaf, ids, teacher)
        (g,) = torch.autograd.grad([r.logprobs, r.entropy, loss], [leaf], [w, w, w])
        return [r.logprobs.detach(), r.entropy.detach(), r.top_ids, r.top_logprobs, loss.detach(), g]

    want = step(new)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(new)
        step(z)
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(z)
    z.copy_(new)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(out, want))
