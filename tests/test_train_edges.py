"""Calls of the training operators at the edges of what they allow, beside the sizes and masks of
tests/test_train_ops.py."""
import threading

import pytest
import torch

import _train_plain as P

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from cresso_b200 import ops as _ops
    return _ops


def _randn(seed, *shape, scale=1.0, dtype=F32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


@gpu
def test_backward_norms_of_host_threads(ops):
    """Calls of one kernel with different stage sizes from several threads at once, each with a stream,
    scratch and outputs of its own: every call is taken, and gives what it gives alone."""
    from cresso_b200 import _lib
    entry = _lib.lib().cresso_block_norm_grad
    code, n = 2, 5  # bfloat16

    def call(width):
        t = [_randn(i, n, width, dtype=BF16) for i in range(4)] + [1 + _randn(4, width, scale=0.1).to(BF16) for _ in "ab"]
        want = ops.block_norm_grad(*t)[:4]
        out = [torch.zeros_like(w) for w in want]
        scratch = torch.empty(ops._scratch_bytes("cresso_block_norm_grad_scratch_bytes", n, width, 0), dtype=torch.uint8,
                              device="cuda")
        stream = torch.cuda.Stream()
        args = (*(x.data_ptr() for x in t), 0, n, width, 0, code, code, code, code, 1.0, 1e-6,
                *(x.data_ptr() for x in out), 0, scratch.data_ptr(), scratch.numel(), stream.cuda_stream)
        return args, out, want, (t, scratch, stream)

    calls = [call(width) for width in (4096, 2048, 1024, 4096)]
    torch.cuda.synchronize()
    errors, start = [], threading.Barrier(len(calls))

    def work(args):
        torch.cuda.set_device(0)
        start.wait()
        for _ in range(20000):
            if entry(*args) != 0:  # the message belongs to the thread
                errors.append(_lib.last_error())
                return

    threads = [threading.Thread(target=work, args=(c[0],)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for _, out, want, _ in calls:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@gpu
@pytest.mark.parametrize("width", [7, 130, 520, 2051, 4096, 4104, 8200, 20001])
@pytest.mark.parametrize("gate_shape", [None, "channel", "full"])
@pytest.mark.parametrize("rd,ad", [(F32, BF16), (F16, F16)])
def test_backward_norm_does_not_read_what_it_does_not_need(ops, width, gate_shape, rd, ad):
    """Without d_y the gradient of the residual is d_h, and d_x has nothing of h; without post_weight d_x
    has nothing of x: infinities, NaN and rows of zeros in them (with eps 0) do not get there."""
    n, inf, nan = 6, float("inf"), float("nan")
    h, x = _randn(1, n, width, dtype=rd), _randn(2, n, width, dtype=ad)
    dh, dy = _randn(3, n, width, dtype=rd), _randn(4, n, width, dtype=ad)
    post, pre = 1 + _randn(5, width, scale=0.2), 1 + _randn(6, width, scale=0.2)
    gate = None if gate_shape is None else _randn(7, *((width,) if gate_shape == "channel" else (n, width)), dtype=ad)
    odd_h, odd_x = h.clone(), x.clone()
    for t in (odd_h, odd_x):
        t[1, width // 2], t[2, 0], t[3], t[5] = inf, nan, 0, -inf
    for args in ((odd_h, x, dh, None, post, pre, gate), (odd_h, x, dh, None, None, None, gate),
                 (odd_h, None, dh, None, None, None, None), (odd_h, odd_x, dh, None, None, pre, gate),
                 (h, odd_x, dh, dy, None, pre, gate), (h, odd_x, None, dy, None, pre, gate)):
        if args[1] is None and rd != ad:
            continue
        want = P.block_norm_grad(*args, 0.35, 0.0)
        got = ops.block_norm_grad(*args, 0.35, 0.0)
        types = (rd, ad, post.dtype, pre.dtype, ad)
        for i, name in enumerate(("d_residual", "d_x", "d_post", "d_pre", "d_gate")):
            present = (True, args[1] is not None, args[4] is not None, args[3] is not None, args[6] is not None)[i]
            assert (got[i] is not None) == present, name
            if present:
                P.check(got[i], *want[i], types[i], name)
        assert torch.isfinite(got[0]).all() and (args[1] is None or torch.isfinite(got[1]).all())


def test_writes_in_place_raise_the_version(ops, monkeypatch):
    """What a call writes counts as changed for autograd, and nothing else does (no GPU: the
    launches are left out)."""
    monkeypatch.setattr(ops, "_train_inputs", lambda what, **tensors: 0)
    monkeypatch.setattr(ops, "_train_call", lambda *args: None)
    logits, ids, teacher = torch.zeros(4, 9), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2)
    ops.distill_grad(logits, ids, teacher)
    ops.distill_loss(logits, ids, teacher)
    assert logits._version == 0
    ops.distill_grad(logits, ids, teacher, inplace=True)
    assert logits._version == 1 and ids._version == teacher._version == 0
    grad, tokens, into = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64), torch.zeros(6, 8)
    ops.embedding_grad(grad, tokens, 6)
    ops.embedding_grad(grad, tokens, 6, into=into)
    assert into._version == 1 and grad._version == tokens._version == 0
    with torch.inference_mode():  # tensors without a version
        logits, into = torch.zeros(4, 9), torch.zeros(6, 8)
        ops.distill_grad(logits, ids, teacher, inplace=True)
        ops.embedding_grad(grad, tokens, 6, into=into)


@gpu
def test_writes_in_place_are_seen_by_autograd(ops):
    """A term that kept the logits, or the tensor that a gradient is added to, for its own backward pass
    gets an error instead of another tensor's values."""
    leaf = _randn(1, 5, 33).requires_grad_()
    logits = leaf * 2
    term = torch.logsumexp(logits, -1).sum()
    with torch.no_grad():
        ops.distill_grad(logits, torch.zeros(5, 2, dtype=torch.int64, device="cuda"), _randn(2, 5, 2), inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        term.backward()
    leaf = _randn(3, 7, 16).requires_grad_()
    into = leaf * 2
    term = into.square().sum()
    with torch.no_grad():
        ops.embedding_grad(_randn(4, 3, 16), torch.tensor([1, 1, 6], device="cuda"), 7, into=into)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        term.backward()


@pytest.mark.parametrize("row0,rows,status", [(2**63 - 1, 2, 1), (2**63 - 5, 10, 1), (2**63 - 1, 2**31 - 256, 1),
                                              (2**63 - 10, 10, 0), (2**63 - 1, 0, 0), (-2**63, 10, 0)])
def test_windows_end_within_64_bits(row0, rows, status):
    """A window whose last row has no 64-bit number would take tokens from the other end of the range."""
    from cresso_b200 import _lib
    lib, p = _lib.lib(), 4096
    # no tokens and nothing to clear: the arguments are checked and nothing is launched
    assert lib.cresso_embedding_gather(p, 0, rows, 8, 8, p, 8, 0, row0, 1.0, p, 0, None) == status
    assert lib.cresso_embedding_grad(p, 0, 0, 8, 8, p, 8, rows, row0, 0, 0, 1.0, p, 0, 1, p, 1 << 20, None) == status


@gpu
def test_last_windows_of_64_bits(ops):
    w = _randn(1, 4, 8)
    tok = torch.tensor([2**63 - 1, -2**63, -2**63 + 1, 2**63 - 4, 2**63 - 5, 0], device="cuda")
    for row0, at in ((2**63 - 4, (3, None, None, 0, None, None)), (-2**63, (None, 0, 1, None, None, None))):
        got = ops.embedding_gather(w, tok, row0=row0)
        grad = ops.embedding_grad(got, tok, 4, row0=row0)
        for i, r in enumerate(at):
            assert torch.equal(got[i], w[r] if r is not None else torch.zeros_like(w[0]))
        for r in range(4):
            assert torch.equal(grad[r], w[r] if r in at else torch.zeros_like(w[0]))
    for row0 in (2**63 - 3, 2**63 - 1):
        with pytest.raises(RuntimeError, match="64 bits"):
            ops.embedding_gather(w, tok, row0=row0)
        with pytest.raises(RuntimeError, match="64 bits"):
            ops.embedding_grad(torch.zeros(6, 8, device="cuda"), tok, 4, row0=row0)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distill_weights_near_the_end_of_the_range(ops, dtype):
    """A logit far above the ones a row begins with, times a weight that is small: the gradient is the
    weight's size, and keeps its digits."""
    n, vocab = 300, 32000
    logits = torch.zeros(n, vocab, dtype=dtype, device="cuda")
    logits[:, 15000] = 39
    logits[1::2, 31999] = 40
    ids, teacher = torch.arange(n, device="cuda")[:, None] + torch.tensor([5, 20000], device="cuda"), _randn(1, n, 2)
    for size in (3e-28, 1e-27, 1e-21, 1e-19, 1e-36):
        weight = torch.full((n,), size, device="cuda")
        weight[::3] *= -1
        (loss, lb), (grad, gb) = P.distill(logits, ids, teacher, weight, 1.5)
        got_loss, got = ops.distill_grad(logits, ids, teacher, weight, 1.5)
        P.check(got_loss, loss, lb, F32, "loss")
        P.check(got, grad, gb, dtype, f"gradient for {size}")


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tau", [0.25, 0.5, 1.0, 4.0])
def test_distill_loss_of_masked_logits(ops, dtype, tau):
    """The teacher's entries on logits of the type's lowest value, one of them or all: probability 0, but a
    finite logit, so the loss is its multiple and not infinite, at temperatures below 1 too."""
    logits, ids, teacher = _randn(1, 6, 1003, dtype=dtype), torch.arange(6 * 4, device="cuda").view(6, 4), _randn(2, 6, 4)
    logits[0, ids[0, 1]] = torch.finfo(dtype).min
    logits[1, ids[1]] = torch.finfo(dtype).min
    logits[2, 30:] = torch.finfo(dtype).min
    logits[3, :30] = torch.finfo(dtype).min
    logits[4, :1000] = torch.finfo(dtype).min
    # the largest loss is weight x temperature x 3.4e38, which has to be a float32 number
    weight = torch.tensor([1.0, 0.25, 1.0, 0.125, -0.25, 1e-30], device="cuda") / max(1.0, tau)
    (loss, lb), (grad, gb) = P.distill(logits, ids, teacher, weight, tau)
    assert torch.isfinite(loss).all() and float(loss.abs().max()) < 3e38
    P.check(ops.distill_loss(logits, ids, teacher, weight, tau), loss, lb, F32, "loss")
    got_loss, got = ops.distill_grad(logits, ids, teacher, weight, tau)
    P.check(got_loss, loss, lb, F32, "loss with gradient")
    P.check(got, grad, gb, dtype, "gradient")
