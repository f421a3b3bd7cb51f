"""GPU: backward passes whose saved tensors come back through saved-tensor hooks -- offloaded to the
host or repacked, so that values are the forward's but strides are not."""
import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

import ltc_cuda

pytestmark = pytest.mark.gpu
B, T, V, H = 4, 6, 37, 12


def normal(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def dense(t):
    return t.clone(memory_format=torch.contiguous_format)


def turned(t):
    """The first two dimensions stored the other way round."""
    return t.transpose(0, 1).contiguous().transpose(0, 1) if t.dim() > 1 else t.clone()


def last_strided(t):
    """Every second element of a buffer twice as long."""
    return torch.stack([t, t], -1)[..., 0]


def padded(t):
    return torch.cat([t, t], -1)[..., :t.shape[-1]] if t.dim() else t.clone()


HOOKS = {
    "offloaded": lambda: save_on_cpu(),
    "offloaded pinned": lambda: save_on_cpu(pin_memory=True),
    **{f.__name__: (lambda f=f: saved_tensors_hooks(lambda t: t, f)) for f in (dense, turned, last_strided, padded)},
}
VIEWS = {
    "shifted": lambda z: z[:, :-1],
    "turned": lambda z: z.transpose(0, 1),
    "every other": lambda z: z[:, ::2],
    "broadcast": lambda z: z[:, :1].expand(B, T, V),
    "whole": lambda z: z,
}


@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("view", VIEWS)
@pytest.mark.parametrize("op", ["distill", "scores"])
def test_vocabulary(op, view, hook):
    base = normal(B, T, V)
    lead = VIEWS[view](base).shape[:-1]
    ids = torch.randint(0, V, (*lead, 3), generator=torch.Generator().manual_seed(1)).cuda()
    weights = normal(*lead, seed=2)

    def grad(ctx=None):
        leaf = base.detach().requires_grad_(True)
        z = VIEWS[view](leaf)

        def forward():
            if op == "distill":
                return ltc_cuda.ltc_distill_loss(z, ids, normal(*lead, 3, seed=3))
            r = ltc_cuda.ltc_token_logprobs(z, ids[..., 0])
            return r.logprobs + 0.5 * r.entropy
        if ctx is None:
            out = forward()
        else:
            with ctx:
                out = forward()
        return torch.autograd.grad([out], [leaf], [weights])[0]

    want = grad()
    got = grad(HOOKS[hook]())
    # the same sums and the same formula an element; a broadcast row's gradient is torch's sum of them
    assert torch.equal(got, want)


@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("op", ["linear", "gated"])
@pytest.mark.parametrize("packed", [False, True])
def test_scans(op, packed, hook):
    """A long scan keeps saved states too; first states, decay and offsets come back as well."""
    n = 2 if op == "linear" else 3
    lead = (200,) if packed else (2, 100)
    base = normal(*lead, n * H, seed=4)
    h0, decay = normal(2, H, seed=5), normal(H, seed=6) - 3
    starts = torch.tensor([0, 90, 200], device="cuda", dtype=torch.int32) if packed else None

    def grad(ctx=None):
        leaves = [t.detach().requires_grad_(True) for t in (base, h0, decay)]
        parts = leaves[0].split(H, dim=-1)
        parts = (torch.tanh(parts[0]), *parts[1:]) if op == "linear" else (*parts, leaves[2])

        def forward():
            fn = ltc_cuda.ltc_linear_scan if op == "linear" else ltc_cuda.ltc_gated_scan
            return fn(*parts, leaves[1], seq_starts=starts)
        if ctx is None:
            outs = forward()
        else:
            with ctx:
                outs = forward()
        wrt = leaves[:2] if op == "linear" else leaves
        return torch.autograd.grad(outs, wrt, [torch.ones_like(o) for o in outs])

    for g, w in zip(grad(HOOKS[hook]()), grad()):
        assert torch.equal(g, w)


def test_another_type_or_shape_is_refused():
    """What a hook does not give back is no operand."""
    z = normal(B, T, V).requires_grad_(True)
    ids = torch.zeros(B, T, 3, dtype=torch.int64, device="cuda")
    x = normal(2, 100, H).requires_grad_(True)
    for change in (lambda t: t.to(torch.bfloat16) if t.is_floating_point() else t,
                   lambda t: t[..., :-1], lambda t: t.cpu()):
        with saved_tensors_hooks(lambda t: t, change):
            outs = [ltc_cuda.ltc_distill_loss(z, ids, normal(B, T, 3)), ltc_cuda.ltc_token_logprobs(z, ids[..., 0])[0],
                    ltc_cuda.ltc_linear_scan(x, x)[0], ltc_cuda.ltc_gated_scan(x, x, x, normal(H))[0]]
        for o, leaf in zip(outs, (z, z, x, x)):
            with pytest.raises(RuntimeError, match="came back"):
                torch.autograd.grad(o.sum(), leaf)


def test_recomputed_in_the_backward():
    """Scan, head and both losses inside a checkpoint: saved tensors are the recomputation's."""
    from torch.utils.checkpoint import checkpoint
    base, head, decay = normal(B, 70, 3 * H, seed=7), normal(H, V, seed=8), normal(H, seed=9) - 3
    ids = torch.randint(0, V, (B, 69, 3), generator=torch.Generator().manual_seed(2)).cuda()
    teacher = normal(B, 69, 3, seed=10)

    def loss(x, w, d):
        h, last = ltc_cuda.ltc_gated_scan(*x.split(H, dim=-1), d)
        z = (h @ w)[:, :-1]
        r = ltc_cuda.ltc_token_logprobs(z, ids[..., 0])
        return ltc_cuda.ltc_distill_loss(z, ids, teacher).sum() + r.entropy.sum() + last.square().sum()

    def grads(run):
        leaves = [t.clone().requires_grad_(True) for t in (base, head, decay)]
        return torch.autograd.grad(run(*leaves), leaves)

    for g, w in zip(grads(lambda *a: checkpoint(loss, *a, use_reentrant=False)), grads(loss)):
        assert torch.equal(g, w)
