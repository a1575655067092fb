"""The C ABI and the argument checks of the training operators, without a GPU: the
library exports what include/cresso_b200_train.h declares, bad arguments come back as
a status before anything is launched, and the Python entry points refuse bad calls."""

import re
from pathlib import Path

import numpy as np
import pytest
import torch

from cresso_b200 import _lib, ops

HEADER = Path(__file__).resolve().parents[1] / "include" / "cresso_b200_train.h"


def test_library_exports_every_declared_symbol():
    lib = _lib.lib()
    names = sorted(re.findall(r"CRESSO_API\s+int\s+(cresso_\w+)\s*\(", HEADER.read_text()))
    assert names == sorted(_lib.TRAIN_EXPORTS)
    for name in names:
        assert hasattr(lib, name), name
    assert int(re.search(r"CRESSO_TRAIN_MAX_TOP = (\d+)", HEADER.read_text()).group(1)) == _lib.TRAIN_MAX_TOP


def _gather(**kw):
    a = dict(weight=4096, wd=0, rows=10, width=8, stride=8, tokens=4096, tb=8, n=4, row0=0, scale=1.0, out=4096, od=0)
    a.update(kw)
    return _lib.lib().cresso_embedding_gather(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(wd=3), 2), (dict(od=3), 2), (dict(wd=-1), 2), (dict(tb=2), 1), (dict(n=-1), 1), (dict(rows=-1), 1),
    (dict(stride=7), 1), (dict(weight=0), 1), (dict(tokens=0), 1), (dict(out=0), 1), (dict(n=2**31), 2),
    (dict(rows=2**31), 2), (dict(n=0, tokens=0, out=0), 0), (dict(width=0, stride=0, out=0), 0)])
def test_gather_status(kw, status):
    assert _gather(**kw) == status, _lib.last_error()


def _egrad(**kw):
    a = dict(grad=4096, gd=0, n=4, width=8, stride=8, tokens=4096, tb=8, rows=10, row0=0, has_padding=0, padding=0,
             scale=1.0, out=4096, od=0, accumulate=0, scratch=4096, nbytes=1 << 20)
    a.update(kw)
    return _lib.lib().cresso_embedding_grad(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(gd=3), 2), (dict(od=9), 2), (dict(tb=1), 1), (dict(stride=7), 1), (dict(n=-1), 1), (dict(rows=-2), 1),
    (dict(n=2**31), 2), (dict(rows=2**31), 2), (dict(out=0), 1), (dict(grad=0), 1), (dict(tokens=0), 1),
    (dict(scratch=0), 4), (dict(nbytes=16), 4), (dict(scratch=4104), 1), (dict(width=4194241, stride=4194241), 2),
    (dict(rows=0, out=0), 0), (dict(width=0, stride=0, out=0), 0),
    (dict(n=0, accumulate=1), 0)])
def test_embedding_grad_status(kw, status):
    assert _egrad(**kw) == status, _lib.last_error()


def test_embedding_grad_scratch_is_host_logic():
    nbytes = np.zeros(1, dtype=np.int64)
    p = nbytes.ctypes.data_as(_lib._pi64)
    assert _lib.lib().cresso_embedding_grad_scratch_bytes(1000, 500, 64, p) == 0
    assert nbytes[0] >= 4 * 1000 + 4 * 501
    assert _lib.lib().cresso_embedding_grad_scratch_bytes(-1, 500, 64, p) == 1
    assert _lib.lib().cresso_embedding_grad_scratch_bytes(1, 500, 64, None) == 1


def _norm(**kw):
    a = dict(residual=4096, x=4096, post=4096, pre=4096, gate=4096, n=6, width=8, gate_rows=3, rd=0, ad=2, wd=0, gd=0,
             scale=1.0, eps=1e-6, h=4096, y=4096)
    a.update(kw)
    return _lib.lib().cresso_block_norm(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(rd=2, ad=0), 2), (dict(rd=2, ad=1), 2), (dict(rd=3, ad=3), 2), (dict(wd=3), 2), (dict(gd=3), 2),
    (dict(n=-1), 1), (dict(width=-1), 1), (dict(gate_rows=4), 1), (dict(gate_rows=0), 1), (dict(eps=-1.0), 1),
    (dict(eps=float("nan")), 1), (dict(x=0), 1), (dict(residual=0), 1), (dict(h=0), 1), (dict(y=0), 1),
    (dict(pre=0), 1), (dict(x=0, post=0, gate=0, pre=0, y=0), 1), (dict(n=2**31, gate=0), 2), (dict(n=2**28, gate=0), 2),
    (dict(width=65537), 2), (dict(n=0), 0),
    (dict(width=0), 0)])
def test_block_norm_status(kw, status):
    assert _norm(**kw) == status, _lib.last_error()


def _ngrad(**kw):
    a = dict(h=4096, x=4096, dh=4096, dy=4096, post=4096, pre=4096, gate=4096, n=6, width=8, gate_rows=3, rd=0, ad=2,
             wd=0, gd=0, scale=1.0, eps=1e-6, dres=4096, dx=4096, dpost=4096, dpre=4096, dgate=4096, scratch=4096,
             nbytes=1 << 24)
    a.update(kw)
    return _lib.lib().cresso_block_norm_grad(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(rd=1, ad=2), 2), (dict(wd=4), 2), (dict(n=-1), 1), (dict(gate_rows=4), 1), (dict(h=0), 1),
    (dict(dres=0), 1), (dict(dh=0, dy=0, dpre=0), 1), (dict(pre=0), 1), (dict(x=0), 1), (dict(dx=0), 1),
    (dict(dpost=0), 1), (dict(dpre=0), 1), (dict(dgate=0), 1), (dict(post=0), 1), (dict(gate=0), 1),
    (dict(scratch=0), 4), (dict(nbytes=8), 4), (dict(scratch=4104), 1), (dict(width=65537), 2), (dict(eps=-1.0), 1),
    (dict(width=0), 0)])
def test_block_norm_grad_status(kw, status):
    assert _ngrad(**kw) == status, _lib.last_error()


def _distill(**kw):
    a = dict(logits=4096, dt=0, n=4, vocab=10, stride=10, ids=4096, ib=8, teacher=4096, td=0, k=3, weight=0, tau=1.0,
             loss=4096, grad=8192)
    a.update(kw)
    return _lib.lib().cresso_distill(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(dt=3), 2), (dict(td=3), 2), (dict(ib=2), 1), (dict(n=-1), 1), (dict(vocab=0), 1), (dict(stride=9), 1),
    (dict(k=-1), 1), (dict(k=1025), 2), (dict(n=2**31), 2), (dict(tau=0.0), 1), (dict(tau=-1.0), 1),
    (dict(tau=float("nan")), 1), (dict(tau=float("inf")), 1), (dict(logits=0), 1), (dict(loss=0), 1),
    (dict(ids=0), 1), (dict(teacher=0), 1), (dict(stride=12, grad=4096), 1), (dict(n=0), 0)])
def test_distill_status(kw, status):
    assert _distill(**kw) == status, _lib.last_error()


def _f(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


IDS = torch.zeros(4, dtype=torch.int64)


@pytest.mark.parametrize("call,message", [
    (lambda: ops.embedding_gather(_f(3, 4), IDS), "CUDA tensor"),
    (lambda: ops.embedding_gather(_f(3), IDS), r"\(rows, width\)"),
    (lambda: ops.embedding_gather(_f(3, 4, dtype=torch.float64), IDS), "float32, float16 or bfloat16"),
    (lambda: ops.embedding_gather(_f(3, 4), IDS, dtype=torch.float64), "float32, float16 or bfloat16"),
    (lambda: ops.embedding_gather(_f(3, 4), _f(4)), "int32 or int64"),
    (lambda: ops.embedding_gather(torch.nn.Parameter(_f(3, 4)), IDS), "not recorded by autograd"),
    (lambda: ops.embedding_grad(_f(3, 4), IDS, 9), r"\*tokens.shape"),
    (lambda: ops.embedding_grad(_f(4, 4), IDS.int().short(), 9), "int32 or int64"),
    (lambda: ops.embedding_grad(_f(4, 4), IDS, -1), "rows must be"),
    (lambda: ops.embedding_grad(_f(4, 4), IDS, 9, into=_f(8, 4)), "into must be"),
    (lambda: ops.embedding_grad(_f(4, 4), IDS, 9, into=_f(4, 9).t()), "into must be"),
    (lambda: ops.embedding_grad(_f(4, 4), IDS, 9, into=_f(9, 4), dtype=torch.float16), "not the type of into"),
    (lambda: ops.embedding_grad(_f(4, 4), IDS, 9, row0=2**63), "64 bits"),
    (lambda: ops.embedding_grad(_f(4, 4), IDS, 9, padding=-2**63 - 1), "64 bits"),
    (lambda: ops.embedding_grad(_f(4, 4), IDS, 9), "CUDA tensor"),
    (lambda: ops.block_norm(_f(2, 4), _f(2, 5)), "x is"),
    (lambda: ops.block_norm(_f(2, 4, dtype=torch.float16), _f(2, 4)), "residual's type"),
    (lambda: ops.block_norm(_f(2, 4), post_weight=_f(4)), "need x"),
    (lambda: ops.block_norm(_f(2, 4), _f(2, 4), _f(5)), "post_weight must be"),
    (lambda: ops.block_norm(_f(2, 4), _f(2, 4), _f(4), _f(4, dtype=torch.float16)), "one type"),
    (lambda: ops.block_norm(_f(2, 3, 4), _f(2, 3, 4), gate=_f(3, 4)), "consecutive rows"),
    (lambda: ops.block_norm(_f(2, 3, 4), _f(2, 3, 4), gate=_f(2, 3, 1)), "consecutive rows"),
    (lambda: ops.block_norm(_f(2, 3, 4), _f(2, 3, 4), gate=_f(2, 2, 3, 4)), "consecutive rows"),
    (lambda: ops.block_norm(_f(2, 4), _f(2, 4), dtype=torch.float16), "y has x's type"),
    (lambda: ops.block_norm(_f(2, 4), _f(2, 4)), "CUDA tensor"),
    (lambda: ops.block_norm_grad(_f(2, 4), _f(2, 4), None, None), "one of d_h and d_y"),
    (lambda: ops.block_norm_grad(_f(2, 4), _f(2, 4), None, _f(2, 4)), "needs pre_weight"),
    (lambda: ops.block_norm_grad(_f(2, 4), _f(2, 4), _f(2, 5), None), "d_h must be"),
    (lambda: ops.block_norm_grad(_f(2, 4), _f(2, 4, dtype=torch.float16), None, _f(2, 4), None, _f(4)), "d_y must be"),
    (lambda: ops.block_norm_grad(_f(2, 4), _f(2, 4), _f(2, 4), None), "CUDA tensor"),
    (lambda: ops.distill_loss(_f(4, 9), IDS[:, None], _f(4, 2)), "same leading shape"),
    (lambda: ops.distill_loss(_f(3, 9), IDS[:, None], _f(4, 1)), "same leading shape"),
    (lambda: ops.distill_loss(_f(4, 9), _f(4, 1), _f(4, 1)), "int32 or int64"),
    (lambda: ops.distill_loss(_f(4, 9), IDS[:, None], _f(4, 1), _f(3)), "weight must be"),
    (lambda: ops.distill_loss(_f(4, 9), IDS[:, None], _f(4, 1), _f(4, dtype=torch.float16)), "weight must be"),
    (lambda: ops.distill_loss(_f(4, 9), torch.zeros(4, 1025, dtype=torch.int64), _f(4, 1025)), "at most 1024"),
    (lambda: ops.distill_grad(_f(9, 4).t(), IDS[:, None], _f(4, 1), inplace=True), "contiguous"),
    (lambda: ops.distill_grad(_f(4, 9).requires_grad_(), IDS[:, None], _f(4, 1)), "not recorded by autograd"),
    (lambda: ops.distill_grad(_f(4, 9), IDS[:, None], _f(4, 1)), "CUDA tensor")])
def test_python_refusals(call, message):
    with pytest.raises(RuntimeError, match=message):
        call()


def test_numbers_are_not_read_from_tensors():
    with pytest.raises(TypeError, match="must be a number"):
        ops.embedding_gather(_f(3, 4), IDS, torch.ones(()))
    with pytest.raises(TypeError, match="must be a number"):
        ops.distill_loss(_f(4, 9), IDS[:, None], _f(4, 1), temperature=torch.ones(()))


def test_calls_run_on_the_tensors_device(monkeypatch):
    """With another device current, an entry point is called with the tensors' device current and
    on that device's current stream."""
    current, seen = [0], []

    class Guard:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *exc):
            current[0] = self.before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 100 + index)

    def entry(*args):
        seen.append((current[0], args))
        return 0

    ops._train_call("x", entry, 0, 7)
    ops._train_call("x", entry, 3, 7, 8)
    assert seen == [(0, (7, 100)), (3, (7, 8, 103))] and current == [0]
    with pytest.raises(RuntimeError, match="invalid argument"):
        ops._train_call("x", lambda *a: 1, 0)
