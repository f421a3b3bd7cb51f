"""The torch binding of the sequence operators: one differentiation, calls from several
threads, the opt-in wait check, and what is not recorded."""
import os
import sys
import threading

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ltc-cuda_b200"))
import ltc_cuda  # noqa: E402

pytestmark = pytest.mark.gpu


def _leaves(*shapes, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).cuda().requires_grad_() for s in shapes]


def _linear(leaves):
    return ltc_cuda.ltc_linear_scan(torch.tanh(leaves[0]), leaves[1])


def _gated(leaves):
    return ltc_cuda.ltc_gated_scan(*leaves)


def _distill(leaves):
    ids = torch.arange(8, device="cuda").reshape(1, 8).expand(5, 8)
    return (ltc_cuda.ltc_distill_loss(leaves[0], ids, torch.zeros(5, 8, device="cuda")),)


def _scores(leaves):
    return ltc_cuda.ltc_token_logprobs(leaves[0], torch.arange(5, device="cuda"))[:2]


CALLS = {
    "linear": (_linear, [(2, 9, 7), (2, 9, 7)]),
    "gated": (_gated, [(2, 9, 7), (2, 9, 7), (2, 9, 7), (7,)]),
    "distill": (_distill, [(5, 33)]),
    "scores": (_scores, [(5, 33)]),
}


def _total(outs):
    return sum(((i + 1) * o.float()).sum() for i, o in enumerate(outs))


@pytest.mark.parametrize("name", CALLS)
def test_differentiable_once(name):
    call, shapes = CALLS[name]
    leaves = _leaves(*shapes)
    plain = torch.autograd.grad(_total(call(leaves)), leaves)
    recorded = torch.autograd.grad(_total(call(leaves)), leaves, create_graph=True)
    assert all(torch.equal(p, r) for p, r in zip(plain, recorded))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        torch.autograd.grad(sum(r.square().sum() for r in recorded), leaves)


@pytest.mark.parametrize("name", CALLS)
def test_nothing_recorded_without_gradients(name):
    call, shapes = CALLS[name]
    leaves = _leaves(*shapes)
    outs = call(leaves)
    assert all(o.requires_grad for o in outs)
    with torch.no_grad():
        again = call(leaves)
    with torch.inference_mode():
        third = call(leaves)
    for o, a, t in zip(outs, again, third):
        assert not a.requires_grad and not t.requires_grad
        assert torch.equal(o.detach(), a) and torch.equal(a, t.clone())


def test_alternatives_carry_no_gradient():
    (z,) = _leaves((5, 33))
    r = ltc_cuda.ltc_token_logprobs(z, torch.arange(5, device="cuda"), top_k=3)
    assert r.logprobs.requires_grad and r.entropy.requires_grad
    assert not r.top_ids.requires_grad and not r.top_logprobs.requires_grad


def test_step_in_place_returns_the_state_given():
    state = torch.zeros(3, 7, device="cuda")
    x = torch.ones(3, 7, device="cuda")
    h, out = ltc_cuda.ltc_gated_scan_step(x, x, x, torch.zeros(7, device="cuda"), state, out_state=state)
    assert out is state and torch.equal(h, state) and bool((state > 0).all())


def test_changed_input_is_noticed():
    x, rate, gate, decay = _leaves((2, 9, 7), (2, 9, 7), (2, 9, 7), (7,))
    h, _ = ltc_cuda.ltc_gated_scan(x, rate, gate, decay)
    with torch.no_grad():
        x += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


@pytest.mark.parametrize("name", CALLS)
def test_threads_on_streams_of_their_own(name):
    call, shapes = CALLS[name]
    want = []
    for i in range(4):
        leaves = _leaves(*shapes, seed=i)
        want.append(torch.autograd.grad(_total(call(leaves)), leaves))
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                leaves = _leaves(*shapes, seed=i)
                for _ in range(20):
                    got[i] = torch.autograd.grad(_total(call(leaves)), leaves)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))


def test_wait_check(monkeypatch):
    x, rate, gate, decay = _leaves((2, 9, 7), (2, 9, 7), (2, 9, 7), (7,))
    ltc_cuda.set_check_waits(True)
    try:
        ltc_cuda.ltc_gated_scan(x, rate, gate, decay)[0].sum().backward()
        monkeypatch.setattr(ltc_cuda, "wait_timeouts", lambda: ltc_cuda._CHECK_WAITS[1] + 2)
        with pytest.raises(RuntimeError, match="scan backward: .* expired"):
            ltc_cuda.ltc_gated_scan(x, rate, gate, decay)[0].sum().backward()
    finally:
        monkeypatch.undo()
        ltc_cuda.set_check_waits(False)
    ltc_cuda.ltc_gated_scan(x, rate, gate, decay)[0].sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_step_operands_that_need_a_copy(dtype):
    """Ordinary operands go straight to the binding; the others give the same through a copy."""
    g = torch.Generator().manual_seed(3)
    x, rate, gate = (torch.randn(5, 12, generator=g).to(dtype).cuda() for _ in range(3))
    decay, state = torch.randn(12, generator=g).cuda(), torch.randn(5, 12, generator=g).cuda()
    want = ltc_cuda.ltc_gated_scan_step(x, rate, gate, decay, state)
    turned = lambda t: t.t().contiguous().t()  # noqa: E731
    spread = torch.stack([decay, decay], 1)[:, 0]
    assert turned(x).stride(-1) != 1 and spread.stride(0) == 2
    for args in ((turned(x), rate, gate, decay, state), (x, rate, turned(gate), decay, state),
                 (x, rate, gate, spread, state), (x, rate, gate, decay, turned(state))):
        assert all(torch.equal(u, v) for u, v in zip(ltc_cuda.ltc_gated_scan_step(*args), want))
    for scale in (8, torch.tensor(8.0).item()):
        got = ltc_cuda.ltc_gated_scan_step(x, rate, gate, decay, state, scale=scale)
        assert all(torch.equal(u, v) for u, v in zip(got, want))


def test_step_refusals_on_the_gpu():
    z = torch.zeros(4, 6, device="cuda")
    d = torch.zeros(6, device="cuda")
    pool = torch.zeros(30, device="cuda")
    step = ltc_cuda.ltc_gated_scan_step
    for exc, args, kw in (
            (TypeError, (z.double(), z, z, d, z), {}), (TypeError, (z, z.bfloat16(), z, d, z), {}),
            (TypeError, (z, z, z, d.half(), z), {}), (ValueError, (z, z[:2], z, d, z), {}),
            (ValueError, (z, z, z, d[:5], z), {}), (ValueError, (z, z, z, d, z.cpu()), {}),
            (ValueError, (z, z, z, d, z[:, :5]), {}), (ValueError, (z, z, z, d, z), dict(scale=0.0)),
            (ValueError, (z, z, z, d, z), dict(scale=float("nan"))),
            (ValueError, (z, z, z, d, z), dict(scale=float("inf"))),
            (ValueError, (z, z, z, d, z), dict(out_state=z.half())),
            (ValueError, (z, z, z, d, z), dict(out_state=torch.zeros(6, 4, device="cuda").t())),
            (ValueError, (z, z, z, d, pool[:24].view(4, 6)), dict(out_state=pool[6:].view(4, 6))),
            (RuntimeError, (z, z, z, d.clone().requires_grad_(), z), {}),
            (TypeError, ([1.0], z, z, d, z), {})):
        with pytest.raises(exc):
            step(*args, **kw)
    assert step(z, z, z, d, z)[0].shape == (4, 6)
