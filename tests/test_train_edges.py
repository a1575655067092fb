"""Calls of the training operators at the edges of what they allow, beside the sizes and masks of
tests/test_train_ops.py."""
import threading

import pytest
import torch

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
