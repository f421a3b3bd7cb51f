"""CPU: what the sequence operators refuse, and the data-parallel steps that call them."""
import ctypes
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import data_parallel
import ltc_cuda


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("exc,fn", [
    (TypeError, lambda: ltc_cuda.ltc_linear_scan([1.0], t(1, 2, 3))),
    (TypeError, lambda: ltc_cuda.ltc_linear_scan(t(1, 2, 3, dtype=torch.float64), t(1, 2, 3, dtype=torch.float64))),
    (TypeError, lambda: ltc_cuda.ltc_linear_scan(t(1, 2, 3), t(1, 2, 3, dtype=torch.bfloat16))),
    (ValueError, lambda: ltc_cuda.ltc_linear_scan(t(2, 3), t(2, 3))),
    (ValueError, lambda: ltc_cuda.ltc_linear_scan(t(1, 2, 3), t(1, 2, 4))),
    (ValueError, lambda: ltc_cuda.ltc_linear_scan(t(1, 2, 3), t(1, 2, 3), t(2, 3))),
    (TypeError, lambda: ltc_cuda.ltc_linear_scan(t(1, 2, 3), t(1, 2, 3), t(1, 3, dtype=torch.float16))),
    (ValueError, lambda: ltc_cuda.ltc_linear_scan(t(1, 2, 3), t(1, 2, 3), seq_starts=t(2, dtype=torch.int32))),
    (ValueError, lambda: ltc_cuda.ltc_linear_scan(t(2, 3), t(2, 3), seq_starts=t(1, dtype=torch.int32))),
    (ValueError, lambda: ltc_cuda.ltc_linear_scan(t(2, 3), t(2, 3), seq_starts=t(2, 2, dtype=torch.int32))),
    (TypeError, lambda: ltc_cuda.ltc_linear_scan(t(2, 3), t(2, 3), seq_starts=t(2))),
    (ValueError, lambda: ltc_cuda.ltc_linear_scan(t(2, 3), t(2, 3), t(2, 3), seq_starts=t(2, dtype=torch.int32))),
    (ValueError, lambda: ltc_cuda.ltc_linear_scan(t(1, 2, 3), t(1, 2, 3))),  # not on a GPU
    (ValueError, lambda: ltc_cuda.ltc_gated_scan(t(1, 2, 3), t(1, 2, 3), t(1, 3, 3), t(3))),
    (ValueError, lambda: ltc_cuda.ltc_gated_scan_step(t(1, 2, 3), t(1, 2, 3), t(1, 2, 3), t(3), t(1, 3))),
    (ValueError, lambda: ltc_cuda.ltc_gated_scan_step(t(2, 3), t(2, 3), t(2, 4), t(3), t(2, 3))),
    (ValueError, lambda: ltc_cuda.ltc_gated_scan_step(t(2, 3), t(2, 3), t(2, 3), t(3), t(2, 3))),
    (TypeError, lambda: ltc_cuda.ltc_distill_loss(t(2, 5, dtype=torch.int64), t(2, 1, dtype=torch.int64), t(2, 1))),
    (ValueError, lambda: ltc_cuda.ltc_distill_loss(t(2, 0), t(2, 1, dtype=torch.int64), t(2, 1))),
    (ValueError, lambda: ltc_cuda.ltc_distill_loss(t(2, 5), t(2, 1, dtype=torch.int64), t(2, 1), temperature=0.0)),
    (ValueError, lambda: ltc_cuda.ltc_distill_loss(t(2, 5), t(2, 1, dtype=torch.int64), t(2, 1), temperature=1e-40)),
    (ValueError, lambda: ltc_cuda.ltc_token_logprobs(t(2, 5), t(2, dtype=torch.int64), temperature=float("nan"))),
    (ValueError, lambda: ltc_cuda.ltc_token_logprobs(t(2, 5), t(2, dtype=torch.int64))),
])
def test_refusals(exc, fn):
    with pytest.raises(exc):
        fn()


def test_refusals_behind_the_device_check(monkeypatch):
    """The remaining argument checks, with the device check taken as passed."""
    monkeypatch.setattr(ltc_cuda, "_on_cuda", lambda *_: None)
    d, i64 = ltc_cuda, torch.int64
    for exc, fn in [
        (ValueError, lambda: d.ltc_gated_scan(t(1, 2, 3), t(1, 2, 3), t(1, 2, 3), t(4))),
        (TypeError, lambda: d.ltc_gated_scan(t(1, 2, 3), t(1, 2, 3), t(1, 2, 3), t(3, dtype=torch.bfloat16))),
        (ValueError, lambda: d.ltc_gated_scan(t(1, 2, 3), t(1, 2, 3), t(1, 2, 3), t(3), scale=0.0)),
        (ValueError, lambda: d.ltc_gated_scan(t(1, 2, 3), t(1, 2, 3), t(1, 2, 3), t(3), scale=float("inf"))),
        (ValueError, lambda: d.ltc_gated_scan_step(t(2, 3), t(2, 3), t(2, 3), t(3), t(2, 4))),
        (ValueError, lambda: d.ltc_gated_scan_step(t(2, 3), t(2, 3), t(2, 3), t(3), t(2, 3), out_state=t(3, 2))),
        (ValueError, lambda: d.ltc_gated_scan_step(t(2, 3), t(2, 3), t(2, 3), t(3), t(2, 3), out_state=t(3, 2).T)),
        (RuntimeError, lambda: d.ltc_gated_scan_step(t(2, 3).requires_grad_(), t(2, 3), t(2, 3), t(3), t(2, 3))),
        (ValueError, lambda: d.ltc_distill_loss(t(2, 5), t(2, 1, dtype=i64), t(3, 1))),
        (ValueError, lambda: d.ltc_distill_loss(t(2, 5), t(2, 257, dtype=i64), t(2, 257))),
        (ValueError, lambda: d.ltc_distill_loss(t(2, 5), t(2, 0, dtype=i64), t(2, 0))),
        (ValueError, lambda: d.ltc_distill_loss(t(2, 5), t(2, 3, dtype=i64), t(2, 2))),
        (TypeError, lambda: d.ltc_distill_loss(t(2, 5), t(2, 2), t(2, 2))),
        (TypeError, lambda: d.ltc_distill_loss(t(2, 5), t(2, 2, dtype=i64), t(2, 2, dtype=i64))),
        (TypeError, lambda: d.ltc_token_logprobs(t(2, 5), t(2))),
        (ValueError, lambda: d.ltc_token_logprobs(t(2, 5), t(3, dtype=i64))),
        (ValueError, lambda: d.ltc_token_logprobs(t(2, 5), t(2, dtype=i64), top_k=6)),
        (ValueError, lambda: d.ltc_token_logprobs(t(2, 500), t(2, dtype=i64), top_k=65)),
        (ValueError, lambda: d.ltc_token_logprobs(t(2, 5), t(2, dtype=i64), top_k=-1)),
    ]:
        with pytest.raises(exc):
            fn()
    buf = t(7)
    with pytest.raises(ValueError, match="overlap"):
        d.ltc_gated_scan_step(t(2, 3), t(2, 3), t(2, 3), t(3), buf[:6].view(2, 3), out_state=buf[1:].view(2, 3))


def test_row_strides_of_logits(monkeypatch):
    """Every view's rows are where the two strides say they are."""
    monkeypatch.setattr(ltc_cuda, "_on_cuda", lambda *_: None)
    base = torch.arange(2 * 3 * 4 * 5, dtype=torch.float32).reshape(2, 3, 4, 5)
    for v in (base, base[:, :, 1:], base[:, 1:], base.transpose(0, 1), base[..., :3], base[0], base[0, 0, 0],
              base[:1].expand(6, 3, 4, 5), base[:, :, :1], base.transpose(2, 3), base[:, ::2, ::2], base[:0]):
        kept, (rows, inner, so, si, V, dt, tau) = ltc_cuda._logits_operand(v, 1.0)
        assert rows == v[..., 0].numel() and V == v.shape[-1] and inner >= 1
        flat, want = kept, v.reshape(-1, V)
        store = torch.as_strided(flat, (flat.untyped_storage().nbytes() // 4 - flat.storage_offset(),), (1,),
                                 flat.storage_offset())
        for r in range(rows):
            at = (r // inner) * so + (r % inner) * si
            assert torch.equal(store[at:at + V], want[r])


def test_c_entries_refuse_without_a_gpu():
    """NULL and out-of-range arguments come back as errors with a message, never as a crash."""
    lib = ltc_cuda._lib
    if lib is None:
        pytest.skip("library not built")
    p = ltc_cuda.LtcScanPlan()
    assert lib.ltc_scan_plan(None, ctypes.byref(p)) != 0
    for bad in ((1, 0x7fff0001, 1, 0, 0), (1, 1, (1 << 28) + 1, 0, 0), (0, 1, 1, 0, 0), (1, 0, 1, 0, 0), (1, 1, 1, 3, 0), (2, 1, 1, 0, 1), (1, 1, 1, 0, -1)):
        assert lib.ltc_scan_plan(ctypes.byref(ltc_cuda.LtcScanDims(*bad)), ctypes.byref(p)) != 0
        assert lib.ltc_last_error()
    assert lib.ltc_gated_scan_step(None, None, None, None, None, 8.0, None, None, None, None) != 0
    assert lib.ltc_token_logprobs_forward(None, None, 0, None, None, None, None, None, None) != 0
    for rows, V, dt, tau in ((0, 5, 0, 1.0), (1, 0, 0, 1.0), (1, 5, 7, 1.0), (1, 5, 0, 0.0), (1, 5, 0, float("nan"))):
        d = ltc_cuda.LtcLogits(16, rows, 1, 0, 5, V, dt, tau)
        assert lib.ltc_distill_forward(ctypes.byref(d), None, None, 0, 1, None, None, None, None) != 0


class _Head(torch.nn.Module):
    def __init__(self):
        super().__init__()
        g = torch.Generator().manual_seed(0)
        self.w = torch.nn.Parameter(torch.randn(4, 11, generator=g))

    def forward(self, x):
        return x @ self.w, None


def _distill(logits, ids, teacher, temperature=1.0):
    lq = torch.log_softmax(logits / temperature, -1).gather(-1, ids)
    p = torch.softmax(teacher / temperature, -1)
    return temperature ** 2 * (p * (p.log() - lq)).sum(-1)


def _scores(logits, tokens, top_k=0, temperature=1.0):
    lq = torch.log_softmax(logits / temperature, -1)
    lp = torch.where(tokens >= 0, lq.gather(-1, tokens.clamp(min=0)[..., None])[..., 0], 0.0)
    return ltc_cuda.TokenLogprobs(lp, -(lq.exp() * lq).sum(-1), None, None)


def _data():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 3, 4, generator=g)
    return x, torch.randint(0, 11, (6, 3, 2), generator=g), torch.randn(6, 3, 2, generator=g), \
        torch.randint(-1, 11, (6, 3), generator=g)


def _steps(lo, hi):
    ltc_cuda.ltc_distill_loss, ltc_cuda.ltc_token_logprobs = _distill, _scores
    x, ids, teacher, tokens = (v[lo:hi] for v in _data())
    m = _Head()
    bucket = data_parallel.FlatGradBucket(m.parameters())
    opt = torch.optim.SGD(m.parameters(), lr=0.1)
    data_parallel.training_step(m, x, bucket, opt, teacher=(ids, teacher), temperature=1.5)
    return bucket.flat.clone(), data_parallel.evaluation_step(m, x, tokens)


def _rank(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    lo, hi = data_parallel.shard_range(6, rank, world)
    grad, sums = _steps(lo, hi)
    if rank == 0:
        q.put((grad.tolist(), sums.tolist()))
    dist.destroy_process_group()


def test_two_ranks_train_and_score_like_one(monkeypatch):
    monkeypatch.setattr(ltc_cuda, "ltc_distill_loss", ltc_cuda.ltc_distill_loss)
    monkeypatch.setattr(ltc_cuda, "ltc_token_logprobs", ltc_cuda.ltc_token_logprobs)
    grad, sums = _steps(0, 6)
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.SimpleQueue()
    mp.spawn(_rank, args=(2, port, q), nprocs=2)
    g2, s2 = q.get()
    assert torch.allclose(torch.tensor(g2), grad, rtol=1e-5, atol=1e-6)
    assert torch.allclose(torch.tensor(s2, dtype=torch.float64), sums, rtol=1e-5)
    assert sums[2] == (_data()[3] >= 0).sum()


def test_missing_binding_is_named(monkeypatch):
    """The solver works without ltc_torch.so; the sequence operators say that it is missing."""
    monkeypatch.setattr(ltc_cuda, "_HAS_CUDA_KERNELS", True)
    monkeypatch.setattr(ltc_cuda, "_torch_binding", None)
    monkeypatch.setattr(ltc_cuda, "_on_cuda", lambda t, name: None)
    for call in (lambda: ltc_cuda.ltc_linear_scan(t(1, 2, 3), t(1, 2, 3)),
                 lambda: ltc_cuda.ltc_gated_scan_step(t(2, 3), t(2, 3), t(2, 3), t(3), t(2, 3)),
                 lambda: ltc_cuda.ltc_distill_loss(t(2, 9), torch.zeros(2, 4, dtype=torch.long), t(2, 4)),
                 lambda: ltc_cuda.ltc_token_logprobs(t(2, 9), torch.zeros(2, dtype=torch.long))):
        with pytest.raises(RuntimeError, match="ltc_torch.so could not be loaded"):
            call()


def test_batch_past_31_bits_is_refused():
    """One more than the kernels' 31-bit count of sequences, and one that wraps to a small number."""
    for n in (1 << 31, (1 << 32) + 5):
        wide = t(1, 1, 1).expand(n, 1, 1)
        with pytest.raises(ValueError, match="sequences"):
            ltc_cuda.ltc_linear_scan(wide, wide)
        rows = t(1, 1).expand(n, 1)
        with pytest.raises(ValueError, match="sequences"):
            ltc_cuda.ltc_gated_scan_step(rows, rows, rows, t(1), rows)
        starts = torch.zeros(1, dtype=torch.int32).expand(n + 1)
        with pytest.raises(ValueError, match="sequences"):
            ltc_cuda.ltc_gated_scan(t(4, 3), t(4, 3), t(4, 3), t(3), seq_starts=starts)
