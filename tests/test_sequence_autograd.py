"""GPU: what autograd has to notice about the sequence operators."""
import pytest
import torch

import ltc_cuda

pytestmark = pytest.mark.gpu


def normal(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def test_step_in_place_is_noticed_by_an_earlier_graph():
    """A first state that a scan keeps for its backward, a final state that a loss keeps, and a
    step that overwrites them."""
    x, decay, state = normal(2, 9, 8), normal(8, seed=1), normal(2, 8, seed=2)
    step = lambda s: ltc_cuda.ltc_gated_scan_step(x[:, 0], x[:, 1], x[:, 2], decay, s, out_state=s)  # noqa: E731
    leaf = x.clone().requires_grad_(True)
    h, last = ltc_cuda.ltc_gated_scan(leaf, leaf, leaf, decay, state)
    step(state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    h, last = ltc_cuda.ltc_gated_scan(leaf, leaf, leaf, decay, state)
    square = last.square().sum()
    with torch.no_grad():
        step(last)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        square.backward()
    before = state._version
    ltc_cuda.ltc_gated_scan_step(x[:, 0], x[:, 1], x[:, 2], decay, state)
    assert state._version == before
    # also where an operand has to be copied first
    turned = x[:, 0].t().contiguous().t()
    ltc_cuda.ltc_gated_scan_step(turned, x[:, 1], x[:, 2], decay, state, out_state=state)
    assert state._version > before


def test_step_into_a_tensor_that_requires_a_gradient_is_refused():
    x, decay = normal(2, 8), normal(8, seed=1)
    state = normal(2, 8, seed=2)
    out = state.clone().requires_grad_(True)
    kept = out.detach().clone()
    for first in (x, x.t().contiguous().t()):
        with pytest.raises(RuntimeError, match="no backward pass"):
            ltc_cuda.ltc_gated_scan_step(first, x, x, decay, state, out_state=out)
    assert torch.equal(out, kept)
    with torch.no_grad():
        ltc_cuda.ltc_gated_scan_step(x, x, x, decay, state, out_state=out)
    assert not torch.equal(out, kept)


def test_step_on_inference_tensors():
    """Updated in place inside inference mode, refused outside it as PyTorch's own operations are."""
    with torch.inference_mode():
        x, decay, state = normal(2, 8), normal(8, seed=1), normal(2, 8, seed=2)
        want = ltc_cuda.ltc_gated_scan_step(x, x, x, decay, state)[1]
        ltc_cuda.ltc_gated_scan_step(x, x, x, decay, state, out_state=state)
        assert torch.equal(state, want)
    with pytest.raises(RuntimeError, match="InferenceMode"):
        ltc_cuda.ltc_gated_scan_step(x, x, x, decay, state, out_state=state)
    assert torch.equal(state, want)


def test_forward_mode_is_refused():
    """No tangent comes out, so none may go in, whether or not gradients are recorded."""
    from torch.autograd import forward_ad
    x, decay, state, z = normal(2, 9, 8), normal(8, seed=1), normal(2, 8, seed=2), normal(4, 33, seed=3)
    ids = torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    calls = [
        lambda d: ltc_cuda.ltc_linear_scan(x, d(x)), lambda d: ltc_cuda.ltc_linear_scan(x, x, d(state)),
        lambda d: ltc_cuda.ltc_gated_scan(x, x, x, d(decay)), lambda d: ltc_cuda.ltc_gated_scan(x, d(x), x, decay),
        lambda d: ltc_cuda.ltc_gated_scan_step(x[:, 0], d(x[:, 0]), x[:, 0], decay, state),
        lambda d: ltc_cuda.ltc_gated_scan_step(x[:, 0], x[:, 0], x[:, 0], decay, d(state)),
        lambda d: ltc_cuda.ltc_distill_loss(d(z), ids, z[:, :2]),
        lambda d: ltc_cuda.ltc_token_logprobs(d(z), ids[:, 0], top_k=2),
    ]
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in calls:
            call(lambda t: t)
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)
        with forward_ad._set_fwd_grad_enabled(False):  # nothing is recorded, as in PyTorch's operations
            calls[0](dual)
