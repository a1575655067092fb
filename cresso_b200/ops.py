"""Op-level entry points.

The first part has the argument meaning of the reference's extension functions
(cresso_cuda/cresso_cuda.cpp:170-196), for tests and for callers that drive single
operators.  The second part are the training operators that make the gradients the
optimizer step reads: ``embedding_gather`` / ``embedding_grad``, ``block_norm`` /
``block_norm_grad`` and ``distill_loss`` / ``distill_grad``.  All of them take CUDA
tensors, allocate their outputs with torch, and run on the current stream.
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Sequence, Tuple

import numpy as np
import torch
from torch import Tensor
from torch.autograd.graph import increment_version

from . import _lib
from ._host import multiscale_frequencies


def _stream(t: Tensor):
    return torch.cuda.current_stream(t.device).cuda_stream


def _need_cuda_f32(t: Tensor, name: str) -> Tensor:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.dtype != torch.float32:
        raise RuntimeError(f"{name} must be float32 (got {t.dtype})")
    return t.contiguous()


def hash_index(shape: Sequence[int], bins: int, salt: int, device, offset: int = 0) -> Tensor:
    """Bin index of every flat index of `shape` (reference _hash_index_tensor, cresso_v5.py:495-516)."""
    n = int(np.prod([int(d) for d in shape])) if len(shape) else 1
    out = torch.empty(n, dtype=torch.int64, device=device)
    _lib.check(_lib.lib().cresso_hash_index(int(offset), n, int(bins), int(salt), _lib.ptr(out), _stream(out)),
               "hash_index")
    return out.view(tuple(int(d) for d in shape))


def hash_reduce_mean(x: Tensor, bins: int, salt: int) -> Tensor:
    """ops.hash_reduce_mean (cresso_cuda.cpp:186)."""
    x = _need_cuda_f32(x, "x")
    out = torch.empty(int(bins), dtype=torch.float32, device=x.device)
    _lib.check(_lib.lib().cresso_hash_reduce_mean(_lib.ptr(x), x.numel(), int(bins), int(salt), _lib.ptr(out),
                                                  _stream(x)), "hash_reduce_mean")
    return out


def hash_gather(values: Tensor, shape: Sequence[int], salt: int) -> Tensor:
    """ops.hash_gather (cresso_cuda.cpp:187)."""
    values = _need_cuda_f32(values, "values")
    shape = tuple(int(d) for d in shape)
    out = torch.empty(shape, dtype=torch.float32, device=values.device)
    _lib.check(_lib.lib().cresso_hash_gather(_lib.ptr(values), values.numel(), out.numel(), int(salt), _lib.ptr(out),
                                             _stream(values)), "hash_gather")
    return out


_WS_CACHE: dict = {}


def basis_workspace(shape: Sequence[int], rank: int, max_frequency: int, device) -> Tensor:
    """Shape workspace of the carrier pack (replaces basis_axis_cache + basis_stats_with_cache)."""
    shape = tuple(int(d) for d in shape)
    key = (str(device), shape, int(rank), int(max_frequency))
    ws = _WS_CACHE.get(key)
    if ws is not None:
        return ws
    L = _lib.lib()
    dims = _lib.i64_array(shape)
    nbytes = np.zeros(1, dtype=np.int64)
    _lib.check(L.cresso_shape_workspace_bytes(len(shape), dims, int(rank), 0, 0, nbytes.ctypes.data_as(_lib._pi64)),
               "shape_workspace_bytes")
    ws = torch.empty(int(nbytes[0]), dtype=torch.uint8, device=device)
    fr = np.ascontiguousarray(np.asarray(multiscale_frequencies(rank, len(shape), max_frequency), dtype=np.int64))
    _lib.check(L.cresso_shape_workspace_init(len(shape), dims, int(rank), fr.ctypes.data_as(_lib._pi64), 0, 0,
                                             _lib.ptr(ws), torch.cuda.current_stream(device).cuda_stream),
               "shape_workspace_init")
    _WS_CACHE[key] = ws
    return ws


def basis_project(x: Tensor, rank: int, max_frequency: int = 5) -> Tuple[Tensor, Tensor]:
    """(mean(x * cos_r), mean(x * sin_r)) for r < rank (ops.basis_project, cresso_cuda.cpp:174)."""
    x = _need_cuda_f32(x, "x")
    ws = basis_workspace(tuple(x.shape), rank, max_frequency, x.device)
    oc = torch.empty(int(rank), dtype=torch.float32, device=x.device)
    os_ = torch.empty(int(rank), dtype=torch.float32, device=x.device)
    _lib.check(_lib.lib().cresso_basis_project(_lib.ptr(x), _lib.ptr(ws), _lib.ptr(oc), _lib.ptr(os_), _stream(x)),
               "basis_project")
    return oc, os_


def basis_reconstruct(cos_coeff: Tensor, sin_coeff: Tensor, shape: Sequence[int], max_frequency: int = 5,
                      gates: Optional[Tensor] = None) -> Tensor:
    """shrink * sum_r g_r (c_r cos_r + s_r sin_r) (ops.basis_reconstruct, cresso_cuda.cpp:177)."""
    cc = _need_cuda_f32(cos_coeff, "cos_coeff")
    cs = _need_cuda_f32(sin_coeff, "sin_coeff")
    rank = cc.numel()
    g = _need_cuda_f32(gates, "gates") if gates is not None else None
    ws = basis_workspace(tuple(shape), rank, max_frequency, cc.device)
    out = torch.empty(tuple(int(d) for d in shape), dtype=torch.float32, device=cc.device)
    _lib.check(_lib.lib().cresso_basis_reconstruct(_lib.ptr(cc), _lib.ptr(cs), _lib.ptr(g), _lib.ptr(ws),
                                                   _lib.ptr(out), _stream(cc)), "basis_reconstruct")
    return out


def instant_axis_metric(rel: Tensor, power: float, coupling: float, eps: float) -> Tensor:
    """Axial current metric of a 1-D / 2-D field (ops.instant_axis_metric_2d, cresso_cuda.cpp:190)."""
    rel = _need_cuda_f32(rel, "rel")
    out = torch.empty_like(rel)
    dims = _lib.i64_array(rel.shape)
    _lib.check(_lib.lib().cresso_instant_axis_metric(_lib.ptr(rel), rel.ndim, dims, float(power), float(coupling),
                                                     float(eps), _lib.ptr(out), _stream(rel)), "instant_axis_metric")
    return out


# ------------------------------------------------------------------ training operators
#
# They compute values and explicit gradients and are not recorded by autograd: call them
# under torch.no_grad(), or from the forward / backward of a torch.autograd.Function.
# Element types are float32, float16 and bfloat16; sums and statistics are float32, and
# each output is rounded once to its type.  The same inputs give the same bits every run.

_TRAIN_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ID_BYTES = {torch.int32: 4, torch.int64: 8}


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the stream's address without the object around it: 2 us less a call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


def _train_dtype(dtype, what: str, name: str) -> int:
    code = _TRAIN_DTYPES.get(dtype)
    if code is None:
        raise RuntimeError(f"{what}: {name} must be float32, float16 or bfloat16 (got {dtype})")
    return code


def _train_inputs(what: str, **tensors) -> int:
    """Index of the one CUDA device of the given tensors (None is skipped); nothing among
    them that autograd would have to record."""
    index, grad = -1, torch.is_grad_enabled()
    for t in tensors.values():
        if t is None:
            continue
        at = t.get_device() if isinstance(t, Tensor) else -2  # -1 on the CPU
        if index == -1:
            index = at
        if at != index or at < 0 or (grad and t.requires_grad):
            break
    else:
        return index
    for name, t in tensors.items():  # which one, and why
        if t is None:
            continue
        if not isinstance(t, Tensor):
            raise TypeError(f"{what}: {name} must be a tensor (got {type(t).__name__})")
        if grad and t.requires_grad:
            raise RuntimeError(f"{what} is not recorded by autograd, and {name} requires a gradient: call it under "
                               f"torch.no_grad() or inside a torch.autograd.Function")
        if not t.is_cuda:
            raise RuntimeError(f"{what}: {name} must be a CUDA tensor")
        if t.get_device() != index:
            raise RuntimeError(f"{what}: {name} is on {t.device}, not on cuda:{index}")
    raise RuntimeError(f"{what}: tensors of one CUDA device are needed")


def _number(value, what: str, name: str) -> float:
    if isinstance(value, Tensor):
        raise TypeError(f"{what}: {name} must be a number, not a tensor")
    return float(value)


def _int64(value, what: str, name: str) -> int:
    value = int(value)
    if not -2**63 <= value < 2**63:
        raise RuntimeError(f"{what}: {name} does not fit 64 bits (got {value})")
    return value


def _row_view(t: Tensor) -> Tuple[Tensor, int, int]:
    """(tensor, number of rows, row stride) of (..., width) with the elements of a row
    adjacent and the rows equally far apart: the tensor itself if it is contiguous or has two
    axes with such strides, else a copy."""
    width = t.shape[-1]
    n = t.numel() // width if width else 0
    if t.is_contiguous():
        return t, n, width
    if t.dim() == 2 and t.stride(0) >= width and (t.stride(1) == 1 or width == 1):
        return t, n, t.stride(0) if n > 1 else width
    return t.contiguous(), n, width


def _address(t: Optional[Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _train_call(what: str, fn, device: int, *args) -> None:
    """One C entry point on the current stream of the tensors' device."""
    if device == torch.cuda.current_device():
        status = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _raw_stream(device))
    if status != 0:
        _lib.check(status, what)


@functools.lru_cache(maxsize=256)
def _scratch_bytes(entry: str, *sizes: int) -> int:
    nbytes = ctypes.c_int64()
    _lib.check(getattr(_lib.lib(), entry)(*sizes, ctypes.byref(nbytes)), entry)
    return nbytes.value


def _train_scratch(entry: str, like: Tensor, *sizes: int) -> Tensor:
    return like.new_empty(_scratch_bytes(entry, *sizes), dtype=torch.uint8)


def embedding_gather(weight: Tensor, tokens: Tensor, scale: float = 1.0, *, row0: int = 0,
                     dtype: Optional[torch.dtype] = None) -> Tensor:
    """Rows ``scale * weight[tokens - row0]`` of shape (*tokens.shape, width).

    ``weight`` (rows, width) is a whole table, or the rows [row0, row0 + rows) of one, as a
    rank of a row-sharded optimizer holds them (cresso_b200.distributed); its rows may lie
    further apart than width.  A token outside those rows gives a row of zeros, so that the
    ranks' results add up to the lookup in the whole table.  tokens: int32 or int64.  The
    result has weight's type unless ``dtype`` names another."""
    if weight.dim() != 2:
        raise RuntimeError(f"embedding_gather: weight must be (rows, width) (got {tuple(weight.shape)})")
    dtype = weight.dtype if dtype is None else dtype
    wd, od = _train_dtype(weight.dtype, "embedding_gather", "weight"), _train_dtype(dtype, "embedding_gather", "dtype")
    if tokens.dtype not in _ID_BYTES:
        raise RuntimeError(f"embedding_gather: tokens must be int32 or int64 (got {tokens.dtype})")
    scale = _number(scale, "embedding_gather", "scale")
    device = _train_inputs("embedding_gather", weight=weight, tokens=tokens)
    rows, width = weight.shape
    weight, _, stride = _row_view(weight)
    tokens = tokens.contiguous()
    out = weight.new_empty((*tokens.shape, width), dtype=dtype)
    _train_call("embedding_gather", _lib.lib().cresso_embedding_gather, device, weight.data_ptr(), wd, rows, width,
                stride, tokens.data_ptr(), _ID_BYTES[tokens.dtype], tokens.numel(), _int64(row0, "embedding_gather", "row0"), scale,
                out.data_ptr(), od)
    return out


def embedding_grad(grad: Tensor, tokens: Tensor, rows: int, scale: float = 1.0, *, row0: int = 0,
                   padding: Optional[int] = None, dtype: Optional[torch.dtype] = None,
                   into: Optional[Tensor] = None) -> Tensor:
    """Gradient (rows, width) of the table of ``embedding_gather`` from the gradient ``grad``
    (*tokens.shape, width) of its result: row r is ``scale`` times the sum of grad over the
    positions whose token is row0 + r, other rows are zero.  Tokens outside
    [row0, row0 + rows) and the token ``padding`` take no part.

    The result has grad's type unless ``dtype`` names another.  With ``into`` (contiguous,
    (rows, width), usually ``param.grad``) the sums are added to it in place, which autograd
    sees as such, rows without a token are not touched, and ``into`` is returned.  A row is
    summed in float32 in a fixed order."""
    if tokens.dtype not in _ID_BYTES:
        raise RuntimeError(f"embedding_grad: tokens must be int32 or int64 (got {tokens.dtype})")
    if grad.dim() < 1 or tuple(grad.shape[:-1]) != tuple(tokens.shape):
        raise RuntimeError(f"embedding_grad: grad must be (*tokens.shape, width) (got {tuple(grad.shape)} for tokens "
                           f"{tuple(tokens.shape)})")
    rows, width = int(rows), grad.shape[-1]
    if rows < 0:
        raise RuntimeError(f"embedding_grad: rows must be >= 0 (got {rows})")
    if into is not None:
        if dtype is not None and dtype is not into.dtype:
            raise RuntimeError(f"embedding_grad: dtype {dtype} is not the type of into ({into.dtype})")
        if tuple(into.shape) != (rows, width) or not into.is_contiguous():
            raise RuntimeError(f"embedding_grad: into must be contiguous ({rows}, {width}) (got {tuple(into.shape)})")
        dtype = into.dtype
    dtype = grad.dtype if dtype is None else dtype
    gd, od = _train_dtype(grad.dtype, "embedding_grad", "grad"), _train_dtype(dtype, "embedding_grad", "dtype")
    scale, row0 = _number(scale, "embedding_grad", "scale"), _int64(row0, "embedding_grad", "row0")
    padding = None if padding is None else _int64(padding, "embedding_grad", "padding")
    device = _train_inputs("embedding_grad", grad=grad, tokens=tokens, into=into)
    grad, _, stride = _row_view(grad)
    tokens = tokens.contiguous()
    n = tokens.numel()
    out = grad.new_empty((rows, width), dtype=dtype) if into is None else into
    L = _lib.lib()
    scratch = _train_scratch("cresso_embedding_grad_scratch_bytes", grad, n, rows, width)
    _train_call("embedding_grad", L.cresso_embedding_grad, device, grad.data_ptr(), gd, n, width, stride,
                tokens.data_ptr(), _ID_BYTES[tokens.dtype], rows, row0, int(padding is not None),
                0 if padding is None else padding, scale, out.data_ptr(), od, int(into is not None),
                scratch.data_ptr(), scratch.numel())
    if into is not None:
        increment_version(into)  # a backward pass that kept it has to see the write
    return out


def _norm_arguments(what: str, residual: Tensor, x: Optional[Tensor], act_dtype, post_weight, pre_weight, gate):
    """Checks of the block norm; returns (rows, width, gate rows, type codes)."""
    if residual.dim() < 1:
        raise RuntimeError(f"{what}: the residual must be (..., width)")
    width = residual.shape[-1]
    rd, ad = _train_dtype(residual.dtype, what, "residual"), _train_dtype(act_dtype, what, "x")
    if rd != ad and rd != 0:
        raise RuntimeError(f"{what}: x must have the residual's type, or 16 bits beside a float32 residual "
                           f"(got {act_dtype} beside {residual.dtype})")
    if x is not None and x.shape != residual.shape:
        raise RuntimeError(f"{what}: x is {tuple(x.shape)}, the residual {tuple(residual.shape)}")
    if x is None and (post_weight is not None or gate is not None):
        raise RuntimeError(f"{what}: post_weight and gate need x")
    wd = 0
    for name, w in (("post_weight", post_weight), ("pre_weight", pre_weight)):
        if w is None:
            continue
        if w.dim() != 1 or w.shape[0] != width:
            raise RuntimeError(f"{what}: {name} must be ({width},) (got {tuple(w.shape)})")
        wd = _train_dtype(w.dtype, what, name)
    if post_weight is not None and pre_weight is not None and post_weight.dtype is not pre_weight.dtype:
        raise RuntimeError(f"{what}: the two weights must have one type")
    gate_rows, gd = 0, 0
    if gate is not None:
        gd = _train_dtype(gate.dtype, what, "gate")
        if gate.dim() == 1 and gate.shape[0] == width:
            return residual.numel() // width if width else 0, width, 1, (rd, ad, wd, gd)
        lead = tuple(residual.shape[:-1])
        g = (1,) * (residual.dim() - gate.dim()) + tuple(gate.shape[:-1])
        shared = len(g)
        while shared and g[shared - 1] == 1:
            shared -= 1
        if gate.dim() < 1 or gate.shape[-1] != width or len(g) != len(lead) or g[:shared] != lead[:shared]:
            raise RuntimeError(f"{what}: gate {tuple(gate.shape)} is not one row of {width} for each group of "
                               f"consecutive rows of {tuple(residual.shape)}")
        gate_rows = math.prod(g)
    return residual.numel() // width if width else 0, width, gate_rows, (rd, ad, wd, gd)


def block_norm(residual: Tensor, x: Optional[Tensor] = None, post_weight: Optional[Tensor] = None,
               pre_weight: Optional[Tensor] = None, gate: Optional[Tensor] = None, scale: float = 1.0,
               eps: float = 1e-6, dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Optional[Tensor]]:
    """The norm after a block with its gate and residual scale, and the norm before the next
    block, in one pass over rows of (..., width)::

        p = x * rsqrt(mean(x^2) + eps) * post_weight        (without post_weight: p = x)
        h = residual + scale * gate * p                      (without gate: 1; without x: h = residual)
        y = h * rsqrt(mean(h^2) + eps) * pre_weight          (without pre_weight: y is None)

    Returns (h, y): h has the residual's type (it is the residual itself without x), y has
    x's type, which is the residual's or 16 bits beside a float32 residual (without x:
    ``dtype``, else the residual's).  y comes from h before its rounding.  ``gate`` is
    (width,), or broadcasts over the last of the residual's leading axes: (batch, 1, width)
    for (batch, length, width), up to the full shape."""
    act = residual.dtype if x is None and dtype is None else dtype if x is None else x.dtype
    if x is not None and dtype is not None and dtype is not x.dtype:
        raise RuntimeError(f"block_norm: y has x's type ({x.dtype}), not {dtype}")
    n, width, gate_rows, (rd, ad, wd, gd) = _norm_arguments("block_norm", residual, x, act, post_weight, pre_weight,
                                                            gate)
    scale, eps = _number(scale, "block_norm", "scale"), _number(eps, "block_norm", "eps")
    device = _train_inputs("block_norm", residual=residual, x=x, post_weight=post_weight, pre_weight=pre_weight,
                           gate=gate)
    given = residual
    residual, x, post_weight, pre_weight, gate = [
        None if t is None else t.contiguous() for t in (residual, x, post_weight, pre_weight, gate)]
    h = given if x is None else torch.empty_like(residual)
    y = None if pre_weight is None else torch.empty_like(residual, dtype=act) if x is None else torch.empty_like(x)
    if x is not None or y is not None:
        _train_call("block_norm", _lib.lib().cresso_block_norm, device, residual.data_ptr(), _address(x),
                    _address(post_weight), _address(pre_weight), _address(gate), n, width, gate_rows, rd, ad, wd, gd,
                    scale, eps, _address(None if x is None else h), _address(y))
    return h, y


def block_norm_grad(h: Tensor, x: Optional[Tensor], d_h: Optional[Tensor], d_y: Optional[Tensor],
                    post_weight: Optional[Tensor] = None, pre_weight: Optional[Tensor] = None,
                    gate: Optional[Tensor] = None, scale: float = 1.0, eps: float = 1e-6):
    """Gradients of ``block_norm`` from its result ``h`` (without x: its residual), its input
    ``x`` and the gradients of h and y (either may be None): the tuple (d_residual, d_x,
    d_post_weight, d_pre_weight, d_gate), each with the type and shape of what it belongs to,
    None where that is None (d_pre_weight also without d_y).  The statistics are formed again
    from h and x.  Sums over rows are float32 in a fixed order."""
    if d_h is None and d_y is None:
        raise RuntimeError("block_norm_grad: one of d_h and d_y is needed")
    act = x.dtype if x is not None else d_y.dtype if d_y is not None else h.dtype
    n, width, gate_rows, (rd, ad, wd, gd) = _norm_arguments("block_norm_grad", h, x, act, post_weight, pre_weight,
                                                            gate)
    if d_y is not None and pre_weight is None:
        raise RuntimeError("block_norm_grad: d_y needs pre_weight")
    for name, t, like in (("d_h", d_h, h.dtype), ("d_y", d_y, act)):
        if t is not None and (t.shape != h.shape or t.dtype is not like):
            raise RuntimeError(f"block_norm_grad: {name} must be {like} {tuple(h.shape)} (got {t.dtype} "
                               f"{tuple(t.shape)})")
    scale, eps = _number(scale, "block_norm_grad", "scale"), _number(eps, "block_norm_grad", "eps")
    device = _train_inputs("block_norm_grad", h=h, x=x, d_h=d_h, d_y=d_y, post_weight=post_weight,
                           pre_weight=pre_weight, gate=gate)
    h, x, d_h, d_y, post_weight, pre_weight, gate = [
        None if t is None else t.contiguous() for t in (h, x, d_h, d_y, post_weight, pre_weight, gate)]
    d_residual = torch.empty_like(h)
    d_x, d_post, d_gate = [None if t is None else torch.empty_like(t) for t in (x, post_weight, gate)]
    d_pre = None if d_y is None else torch.empty_like(pre_weight)
    L = _lib.lib()
    scratch = _train_scratch("cresso_block_norm_grad_scratch_bytes", h, n, width, gate_rows)
    _train_call("block_norm_grad", L.cresso_block_norm_grad, device, h.data_ptr(), _address(x), _address(d_h),
                _address(d_y), _address(post_weight), _address(pre_weight), _address(gate), n, width, gate_rows, rd,
                ad, wd, gd, scale, eps, d_residual.data_ptr(), _address(d_x), _address(d_post), _address(d_pre),
                _address(d_gate), scratch.data_ptr(), scratch.numel())
    return d_residual, d_x, d_post, d_pre, d_gate


def _distill(what: str, logits: Tensor, ids: Tensor, teacher: Tensor, weight: Optional[Tensor], temperature: float,
             backward: bool, inplace: bool):
    ld, td = _train_dtype(logits.dtype, what, "logits"), _train_dtype(teacher.dtype, what, "teacher")
    if ids.dtype not in _ID_BYTES:
        raise RuntimeError(f"{what}: ids must be int32 or int64 (got {ids.dtype})")
    if logits.dim() < 1 or ids.dim() < 1 or ids.shape[:-1] != logits.shape[:-1] or teacher.shape != ids.shape:
        raise RuntimeError(f"{what}: logits (..., vocab) and ids, teacher (..., k) must have the same leading shape "
                           f"(got {tuple(logits.shape)}, {tuple(ids.shape)}, {tuple(teacher.shape)})")
    if weight is not None and (weight.dtype is not torch.float32 or weight.shape != logits.shape[:-1]):
        raise RuntimeError(f"{what}: weight must be float32 {tuple(logits.shape[:-1])} (got {weight.dtype} "
                           f"{tuple(weight.shape)})")
    if ids.shape[-1] > _lib.TRAIN_MAX_TOP:
        raise RuntimeError(f"{what}: at most {_lib.TRAIN_MAX_TOP} teacher entries in a row (got {ids.shape[-1]})")
    temperature = _number(temperature, what, "temperature")
    if inplace and not logits.is_contiguous():
        raise RuntimeError(f"{what}: inplace needs contiguous logits")
    device = _train_inputs(what, logits=logits, ids=ids, teacher=teacher, weight=weight)
    vocab, k = logits.shape[-1], ids.shape[-1]
    lead = logits.shape[:-1]
    n = math.prod(lead)
    rows, _, stride = _row_view(logits)
    ids, teacher, weight = ids.contiguous(), teacher.contiguous(), None if weight is None else weight.contiguous()
    loss = logits.new_empty(lead, dtype=torch.float32)
    grad = None if not backward else logits if inplace else logits.new_empty(logits.shape)
    _train_call(what, _lib.lib().cresso_distill, device, rows.data_ptr(), ld, n, vocab, stride, ids.data_ptr(),
                _ID_BYTES[ids.dtype], teacher.data_ptr(), td, k, _address(weight), temperature, loss.data_ptr(),
                _address(grad))
    if inplace:
        increment_version(logits)  # a backward pass that kept them has to see the write
    return loss, grad


def distill_loss(logits: Tensor, ids: Tensor, teacher: Tensor, weight: Optional[Tensor] = None,
                 temperature: float = 1.0) -> Tensor:
    """Distillation loss of each row of student logits (..., vocab) from the teacher's top
    logits: ``teacher`` (..., k) at the vocabulary indices ``ids`` (..., k)::

        p = softmax(teacher / temperature) over the row's valid entries
        loss = weight * temperature^2 * sum_k p_k (log p_k - log softmax(logits / temperature)[ids_k])

    An entry is valid when 0 <= id < vocab and its logit is not -inf (pad short lists with
    id -1).  A row with weight 0, or without a valid entry, has loss 0 whatever its logits
    hold.  A row whose student has a logit of -inf at a teacher's entry has loss +inf.  weight:
    float32 of the leading shape, 1 when omitted; the loss is float32."""
    return _distill("distill_loss", logits, ids, teacher, weight, temperature, False, False)[0]


def distill_grad(logits: Tensor, ids: Tensor, teacher: Tensor, weight: Optional[Tensor] = None,
                 temperature: float = 1.0, *, inplace: bool = False) -> Tuple[Tensor, Tensor]:
    """(loss, gradient) of ``distill_loss``: the gradient of the sum of the rows' losses with
    respect to the logits, in their type and shape::

        grad_v = weight * temperature * (softmax(logits / temperature)_v - sum of p_k with id_k = v)

    An id may occur more than once.  ``weight`` carries the mean over the batch and a loss
    scale.  With ``inplace`` the gradient takes the place of the (contiguous) logits, which
    autograd sees as a write to them."""
    return _distill("distill_grad", logits, ids, teacher, weight, temperature, True, inplace)
