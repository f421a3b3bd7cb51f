"""GPU: the sequence operators as they are used together -- a recurrent student over packed or
padded tokens, trained on a teacher's best logits and scored."""
import pytest
import torch

import data_parallel
import ltc_cuda
import ltc_layer

pytestmark = pytest.mark.gpu
D, H, V = 12, 24, 501


class Student(torch.nn.Module):
    """Token embedding, one projection to (x, rate, gate), the scan, a head over the vocabulary."""

    def __init__(self, dtype=torch.float32):
        super().__init__()
        g = torch.Generator().manual_seed(0)
        p = lambda *s, k=1.0: torch.nn.Parameter((torch.randn(*s, generator=g) * k).to(dtype))  # noqa: E731
        self.emb, self.proj, self.head = p(V, D), p(D, 3 * H, k=0.5), p(H, V, k=0.3)
        self.decay = torch.nn.Parameter(torch.randn(H, generator=g) - 3)

    def forward(self, tokens, state=None, seq_starts=None):
        x, rate, gate = (self.emb[tokens] @ self.proj).split(H, dim=-1)
        h, state = ltc_cuda.ltc_gated_scan(x, rate, gate, self.decay, state, seq_starts=seq_starts)
        return h @ self.head, state

    def step(self, tokens, state):
        with torch.no_grad():
            x, rate, gate = (self.emb[tokens] @ self.proj).split(H, dim=-1)
            h, state = ltc_cuda.ltc_gated_scan_step(x, rate, gate, self.decay, state, out_state=state)
            return h @ self.head


def plain_loss(m, tokens, ids, teacher, tau):
    """The same student in fp64 torch operations."""
    x, rate, gate = (m.emb[tokens] @ m.proj).split(H, dim=-1)
    L = -8 * torch.nn.functional.softplus(m.decay) * torch.sigmoid(rate)
    a, b = L.exp(), (-torch.expm1(2 * L)).sqrt() * torch.sigmoid(gate) * x
    h, hs = torch.zeros_like(a[:, 0]), []
    for t in range(a.shape[1]):
        h = a[:, t] * h + b[:, t]
        hs.append(h)
    lq = torch.log_softmax(torch.stack(hs, 1) @ m.head / tau, -1)
    p = torch.softmax(teacher / tau, -1)
    return tau * tau * (p * (p.log() - lq.gather(-1, ids))).sum()


def batch(B=3, T=70):
    g = torch.Generator().manual_seed(3)
    return (torch.randint(0, V, (B, T), generator=g).cuda(), torch.randint(0, V, (B, T, 6), generator=g).cuda(),
            torch.randn(B, T, 6, generator=g).cuda())


def test_training_step_gradients(monkeypatch):
    """training_step with a teacher against fp64 autograd.  fp32 end to end (torch products
    without reduced precision): a few hundred roundings of terms that share the gradient's
    scale, 1e-4 of its largest value allowed."""
    monkeypatch.setattr(torch.backends.cuda.matmul, "allow_tf32", False)
    tokens, ids, teacher = batch()
    m = Student().cuda()
    ref = Student().cuda().double()
    want = plain_loss(ref, tokens, ids, teacher.double(), 1.5)
    grads = torch.autograd.grad(want, list(ref.parameters()))
    bucket = data_parallel.FlatGradBucket(m.parameters())
    loss = data_parallel.training_step(m, tokens, bucket, torch.optim.SGD(m.parameters(), lr=0.0),
                                       teacher=(ids, teacher), temperature=1.5)
    bucket.check_views()
    assert abs(loss.item() - want.item()) < 1e-4 * abs(want.item())
    for p, g in zip(m.parameters(), grads):
        assert (p.grad.double() - g).abs().max() <= 1e-4 * g.abs().max()


def test_packed_equals_padded_and_decoding_continues():
    m = Student().cuda()
    tokens, _, _ = batch(2, 70)
    with torch.no_grad():
        padded, last = m(tokens)
        starts = torch.tensor([0, 70, 110], device="cuda")
        packed, plast = m(torch.cat([tokens[0], tokens[1, :40]]), seq_starts=starts)
        assert torch.allclose(packed[:70], padded[0], rtol=1e-4, atol=1e-5)
        assert torch.allclose(packed[70:], padded[1, :40], rtol=1e-4, atol=1e-5)
        state = plast.clone()
        state[0] = last[0]
        nxt = tokens[:, 40]
        logits = m.step(nxt, state)
    assert torch.allclose(logits[1], padded[1, 40], rtol=1e-4, atol=1e-5)
    r = ltc_cuda.ltc_token_logprobs(logits, nxt, top_k=3)
    assert torch.equal(r.top_ids[:, 0], logits.argmax(-1))


def test_evaluation_step():
    m = Student().cuda()
    tokens, _, _ = batch()
    target = tokens.roll(-1, 1)
    target[:, -1] = -1
    s = data_parallel.evaluation_step(m, tokens, target)
    lq = torch.log_softmax(m(tokens)[0].double(), -1)
    lp = lq.gather(-1, target.clamp(min=0)[..., None])[..., 0]
    given = target >= 0
    assert s[2] == given.sum()
    assert abs(s[0] - lp[given].sum()) < 1e-4 * abs(s[0])
    assert abs(s[1] + (lq.exp() * lq).sum(-1)[given].sum()) < 1e-4 * s[1]


def test_solver_layer_as_student():
    """The solver's layer with a head, trained through the same step: runs and moves its weights."""

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.rnn, self.head = ltc_layer.TrueLiquidTimeConstant(D, H), torch.nn.Linear(H, V)

        def forward(self, x):
            h, state = self.rnn(x)
            return self.head(h), state

    torch.manual_seed(0)
    net = Net().cuda()
    _, ids, teacher = batch(3, 5)
    x = torch.randn(3, 5, D, device="cuda")
    bucket = data_parallel.FlatGradBucket(net.parameters())
    before = net.head.weight.detach().clone()
    loss = data_parallel.training_step(net, x, bucket, torch.optim.SGD(net.parameters(), lr=0.1), teacher=(ids, teacher))
    assert torch.isfinite(loss) and torch.isfinite(bucket.flat).all() and not torch.equal(before, net.head.weight)


def test_captured_training_step_replays():
    """Scan, head and both losses captured into one graph, replayed on another batch."""
    m = Student(torch.bfloat16).cuda()
    tokens, ids, teacher = batch()
    t2, i2, l2 = (v.flip(0).clone() for v in (tokens, ids, teacher))
    params = list(m.parameters())

    def step():
        logits, _ = m(tokens)
        loss = ltc_cuda.ltc_distill_loss(logits, ids, teacher).sum()
        loss = loss - 0.01 * ltc_cuda.ltc_token_logprobs(logits, tokens).entropy.sum()
        return [loss.detach(), *torch.autograd.grad(loss, params)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    tokens.copy_(t2), ids.copy_(i2), teacher.copy_(l2)
    graph.replay()
    torch.cuda.synchronize()
    eager = step()
    # the loss and the decay gradient pass no atomics; the embedding's gradient may (torch)
    assert torch.equal(out[0], eager[0])
    for u, v in zip(out[1:], eager[1:]):
        assert torch.allclose(u.float(), v.float(), rtol=2e-2, atol=2e-2 * v.float().abs().max().item())
