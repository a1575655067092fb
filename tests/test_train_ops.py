"""The training operators on the GPU against their formulas in float64
(tests/_train_plain.py, which derives the bounds)."""

import pytest
import torch

import _train_plain as P

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from cresso_b200 import ops as _ops
    return _ops


def _randn(seed, *shape, scale=1.0, dtype=F32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _tokens(seed, n, rows, dtype=torch.int64, low=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(low, rows, (n,) if isinstance(n, int) else n, generator=gen, device="cuda").to(dtype)


# ---------------------------------------------------------------------------- embedding

SIZES = [(0, 5, 8), (1, 1, 1), (1, 32, 4096), (7, 3, 13), (33, 9, 2050), (257, 31, 64), (1000, 500, 1030),
         (4097, 2000, 96), (513, 1, 40), (300, 149, 24), (65, 5000, 4104)]


@pytest.mark.parametrize("n,rows,width", SIZES)
@pytest.mark.parametrize("wd,od", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16), (BF16, F32), (F32, F16)])
def test_gather(ops, n, rows, width, wd, od):
    w, tok = _randn(1, rows, width, dtype=wd), _tokens(2, n, rows)
    value, bound = P.gather(w, tok, 1.7, 0, od)
    P.check(ops.embedding_gather(w, tok, 1.7, dtype=od), value, bound, od)


def test_gather_window_strides_and_shapes(ops):
    table = _randn(3, 40, 72, dtype=BF16)
    tok = _tokens(4, (3, 11), 50, torch.int32, low=-4)
    for w in (table, table[:, :64], table[:, 8:72], table[:, 1:10], table[::2], table.t(), table[5:6], table[:, 3:4]):
        value, bound = P.gather(w, tok, 0.5, 6, BF16)
        P.check(ops.embedding_gather(w, tok, 0.5, row0=6), value, bound, BF16, str(w.stride()))
    # positions in any order, and row blocks of one table that add up to the whole lookup
    w = table.float()
    value, bound = P.gather(w, tok.t(), 0.5, 0, F32)
    whole = ops.embedding_gather(w, tok.t(), 0.5)
    P.check(whole, value, bound, F32)
    parts = ops.embedding_gather(w[:17], tok.t(), 0.5) + ops.embedding_gather(w[17:], tok.t(), 0.5, row0=17)
    assert torch.equal(parts, whole)


def test_gather_far_ids_and_empty_tables(ops):
    w = _randn(5, 4, 8)
    tok = torch.tensor([0, 3, 4, -1, 2**31 + 1, -2**31, 2**62, -2**62, 2**32], device="cuda")
    value, bound = P.gather(w, tok, 1.0, 0, F32)
    P.check(ops.embedding_gather(w, tok), value, bound, F32)
    assert torch.equal(ops.embedding_gather(w[:0], tok), torch.zeros(9, 8, device="cuda"))
    assert ops.embedding_gather(w[:, :0], tok).shape == (9, 0)
    value, bound = P.gather(w, tok, 1.0, 2**32 - 1, F32)
    P.check(ops.embedding_gather(w, tok, row0=2**32 - 1), value, bound, F32)


@pytest.mark.parametrize("n,rows,width", SIZES)
@pytest.mark.parametrize("gd,od", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16), (F16, F32)])
def test_embedding_grad(ops, n, rows, width, gd, od):
    g, tok = _randn(6, n, width, dtype=gd), _tokens(7, n, rows)
    value, bound = P.embedding_grad(g, tok, rows, 1.7)
    got = ops.embedding_grad(g, tok, rows, 1.7, dtype=od)
    P.check(got, value, bound, od)
    assert torch.equal(got, ops.embedding_grad(g, tok, rows, 1.7, dtype=od))
    into = _randn(8, rows, width, dtype=od)
    before = into.clone()
    value, bound = P.embedding_grad(g, tok, rows, 1.7, into=into)
    assert ops.embedding_grad(g, tok, rows, 1.7, into=into) is into
    P.check(into, value, bound, od)
    untouched = torch.ones(rows, dtype=torch.bool, device="cuda")
    untouched[tok] = False
    assert torch.equal(into[untouched], before[untouched])


@pytest.mark.parametrize("rows,width,n", [(32000, 64, 16384), (1000, 512, 20000), (3, 1024, 9000), (100000, 16, 70000),
                                          (250001, 8, 5000), (174720, 8, 2000), (47000, 8, 16384)])
def test_embedding_grad_uneven_rows(ops, rows, width, n):
    """Most positions fall on a few rows (a frequent word, padding), some on no row at all."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    tok = ((rows + 2.0) ** u - 1).long()  # log-uniform: half of them below sqrt(rows); some at rows and above
    tok[n // 3:n // 2] = rows // 2
    tok[::7] = -100
    g = _randn(10, n, width, dtype=BF16)
    for padding in (None, rows // 2):
        value, bound = P.embedding_grad(g, tok, rows, 1.0, padding=padding)
        got = ops.embedding_grad(g, tok, rows, dtype=F32, padding=padding)
        P.check(got, value, bound, F32)
        assert torch.equal(got, ops.embedding_grad(g, tok, rows, dtype=F32, padding=padding))
    value, bound = P.embedding_grad(g, tok, rows // 3, 1.0, row0=rows // 3)
    P.check(ops.embedding_grad(g, tok, rows // 3, row0=rows // 3, dtype=F32), value, bound, F32)


@pytest.mark.parametrize("rows,width,n", [(400, 128, 131072), (400, 129, 131072), (3000, 9, 200001), (60, 3, 1048577)])
def test_embedding_grad_many_tokens(ops, rows, width, n):
    """Rows that span many tiles, at the bounds of the tiles' sizes."""
    gen = torch.Generator(device="cuda").manual_seed(19)
    tok = (torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) ** 3 * rows).long()
    g = _randn(21, n, width, dtype=F16)
    value, bound = P.embedding_grad(g, tok, rows, 1.0)
    P.check(ops.embedding_grad(g, tok, rows, dtype=F32), value, bound, F32)


def test_embedding_grad_strides_and_ids(ops):
    tok = _tokens(11, (5, 13), 60, torch.int32, low=-5)
    base = _randn(12, 65, 80, dtype=F16)
    for g in (base[:, :64], base[:, 8:72], base[:, 1:10], base[:, 3:4], base[:1].expand(65, 80)):
        value, bound = P.embedding_grad(g, tok, 40, 0.5, row0=6)
        P.check(ops.embedding_grad(g, tok.reshape(-1), 40, 0.5, row0=6), value, bound, F16, str(g.stride()))
    wide = base.reshape(5, 13, 80).transpose(0, 1)
    value, bound = P.embedding_grad(wide, tok.t(), 40, 0.5, row0=6)
    P.check(ops.embedding_grad(wide, tok.t(), 40, 0.5, row0=6), value, bound, F16)
    far = torch.tensor([0, 2**62, -2**62, 2**32, 3, 3], device="cuda")
    g = _randn(13, 6, 8)
    value, bound = P.embedding_grad(g, far, 4, 1.0)
    P.check(ops.embedding_grad(g, far, 4), value, bound, F32)
    assert ops.embedding_grad(g, far, 0).shape == (0, 8)


@pytest.mark.parametrize("width", [1, 2, 7, 8, 9, 33, 130, 515, 2050, 2051, 4095])
@pytest.mark.parametrize("gd,od", [(BF16, BF16), (F16, F32), (F32, BF16), (F32, F32)])
def test_embedding_odd_addresses(ops, width, gd, od):
    """Gradients and tables that only their type aligns, with gaps between the rows: what lies
    around them is NaN, and the bytes around the result stay."""
    n, rows, first = 700, 90, 3
    flat = torch.full((n * (width + 1) + 16,), float("nan"), dtype=gd, device="cuda")
    tok = _tokens(18, n, 60)
    for offset, stride in ((1, width), (5, width + 1), (0, width)):
        flat.fill_(float("nan"))
        g = flat[offset:offset + n * stride].view(n, stride)[:, :width]
        g.copy_(_randn(19, n, width, dtype=gd))
        value, bound = P.embedding_grad(g, tok, rows, 0.5)
        P.check(ops.embedding_grad(g, tok, rows, 0.5, dtype=od), value, bound, od)
        value, bound = P.gather(g, tok, 0.5, 0, od)
        P.check(ops.embedding_gather(g, tok, 0.5, dtype=od), value, bound, od)
        around = torch.full((rows * width + 16,), 7.0, dtype=od, device="cuda")
        into = around[first:first + rows * width].view(rows, width)
        into.copy_(_randn(20, rows, width, dtype=od))
        value, bound = P.embedding_grad(g, tok, rows, 0.5, into=into)
        ops.embedding_grad(g, tok, rows, 0.5, into=into)
        P.check(into, value, bound, od)
        assert (around[:first] == 7).all() and (around[first + rows * width:] == 7).all()


def test_embedding_rows_beyond_32_bit_offsets(ops):
    rows, width = 530001, 4104  # 2.17e9 elements
    w = torch.zeros(rows, width, dtype=BF16, device="cuda")
    w[-3:] = _randn(14, 3, width, dtype=BF16)
    tok = torch.tensor([rows - 1, rows - 3, rows - 2, 0], device="cuda")
    value, bound = P.gather(w[-3:], tok, 2.0, rows - 3, BF16)
    P.check(ops.embedding_gather(w, tok, 2.0), value, bound, BF16)
    del w
    g = _randn(15, 4, width, dtype=BF16)
    got = ops.embedding_grad(g, tok, rows, 2.0)
    value, bound = P.embedding_grad(g, tok, 3, 2.0, row0=rows - 3)
    P.check(got[-3:], value, bound, BF16)
    assert not got[1:-3].any()
    value, bound = P.embedding_grad(g, tok, 1, 2.0)
    P.check(got[:1], value, bound, BF16)


def test_embedding_infinities_stay_in_their_rows(ops):
    w = _randn(16, 4, 24)
    w[1], w[2, 3] = float("nan"), float("inf")
    got = ops.embedding_gather(w, torch.tensor([0, 1, 2, 9], device="cuda"))
    assert torch.isfinite(got[0]).all() and torch.isnan(got[1]).all() and torch.isinf(got[2]).sum() == 1
    assert not got[3].any()
    g = _randn(17, 5, 24)
    g[3] = float("nan")
    tok = torch.tensor([0, 1, 1, 7, 2], device="cuda")
    assert torch.isfinite(ops.embedding_grad(g, tok, 4)).all()  # the NaN row's token is outside
    assert torch.isnan(ops.embedding_grad(g, tok, 8)).sum() == 24


# ---------------------------------------------------------------------------- block norm

NORM_SIZES = [(1, 1, 1), (1, 1, 4096), (2, 3, 7), (3, 5, 64), (2, 33, 250), (3, 341, 130), (1, 9, 2050), (5, 1, 1024),
              (1, 7, 8200), (2, 2, 20001), (4, 64, 512), (1, 2, 40000), (2, 700, 32), (2, 600, 4096), (3, 400, 2560),
              (1, 1201, 1030), (2, 600, 5001), (1, 1190, 520)]
PAIRS = [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16), (F32, F16)]


def _norm_inputs(shape, rd, ad, gate, wd=F32):
    b, n, d = shape
    res, x = _randn(20, *shape, scale=2.0, dtype=rd), _randn(21, *shape, scale=0.7, dtype=ad)
    post, pre = (1 + _randn(22, d, scale=0.3)).to(wd), (1 + _randn(23, d, scale=0.3)).to(wd)
    gs = {"none": None, "channel": (d,), "sample": (b, 1, d), "full": shape}[gate]
    return res, x, post, pre, None if gs is None else _randn(24, *gs, scale=0.5, dtype=ad)


def _check_norm(ops, res, x, post, pre, gate, scale=0.35, eps=1e-6):
    h, y = ops.block_norm(res, x, post, pre, gate, scale, eps)
    want_h, want_y = P.block_norm(res, x, post, pre, gate, scale, eps)
    if x is None:
        assert h is res
    else:
        P.check(h, *want_h, res.dtype, "h")
    if pre is None:
        assert y is None
    else:
        P.check(y, *want_y, res.dtype if x is None else x.dtype, "y")


def _check_norm_grad(ops, res, x, post, pre, gate, scale=0.35, eps=1e-6, dh=True, dy=True):
    ad = res.dtype if x is None else x.dtype
    dh = _randn(25, *res.shape, scale=0.5, dtype=res.dtype) if dh else None
    dy = _randn(26, *res.shape, scale=0.5, dtype=ad) if dy else None
    got = ops.block_norm_grad(res, x, dh, dy, post, pre, gate, scale, eps)
    want = P.block_norm_grad(res, x, dh, dy, post, pre, gate, scale, eps)
    like = (res, x, post, pre if dy is not None else None, gate)
    for name, g, w, t in zip(("d_residual", "d_x", "d_post", "d_pre", "d_gate"), got, want, like):
        assert (g is None) == (t is None), name
        if t is not None:
            P.check(g, *w, t.dtype, name)
    again = ops.block_norm_grad(res, x, dh, dy, post, pre, gate, scale, eps)
    for a, b in zip(got, again):
        assert a is None or torch.equal(a, b)


@pytest.mark.parametrize("shape", NORM_SIZES)
@pytest.mark.parametrize("rd,ad", PAIRS)
@pytest.mark.parametrize("gate", ["none", "channel", "sample", "full"])
def test_block_norm(ops, shape, rd, ad, gate):
    a = _norm_inputs(shape, rd, ad, gate)
    _check_norm(ops, *a)
    _check_norm_grad(ops, *a)


@pytest.mark.parametrize("wd", [F32, F16, BF16])
def test_block_norm_parts(ops, wd):
    """Without each of its parts, and with each type of the weights."""
    res, x, post, pre, gate = _norm_inputs((2, 19, 136), F32, BF16, "sample", wd)
    for a in ((res, x, None, pre, gate), (res, x, post, None, gate), (res, x, None, None, None),
              (res, x, None, pre, None), (res, None, None, pre, None), (res, x, post, pre, gate)):
        _check_norm(ops, *a)
        for dh, dy in ((True, True), (True, False), (False, True)):
            if not (dy and a[3] is None):
                _check_norm_grad(ops, *a, dh=dh, dy=dy)
    h, y = ops.block_norm(res, pre_weight=pre, dtype=BF16)
    assert h is res
    P.check(y, *P.block_norm(res, None, None, pre, None, 1.0, 1e-6)[1], BF16)
    h, y = ops.block_norm(res)
    assert h is res and y is None


def test_block_norm_strides(ops):
    res, x, post, pre, gate = _norm_inputs((6, 10, 64), BF16, BF16, "channel")
    odd = _randn(27, 6, 10, 65, dtype=BF16)
    for r, v in ((res.transpose(0, 1), x.transpose(0, 1)), (odd[..., 1:], x), (res, odd[..., :64]),
                 (res[::2], x[1::2]), (res[:, 1:], x[:, :9]), (res, x[:1].expand(6, 10, 64))):
        _check_norm(ops, r, v, post, pre, gate)
        _check_norm_grad(ops, r, v, post, pre, gate)
    w = _randn(28, 130)
    _check_norm(ops, res, x, w[1:65], w[::2][:64], gate)          # weights at odd addresses and strides
    _check_norm_grad(ops, res, x, w[1:65], w[::2][:64], gate[:])


@pytest.mark.parametrize("n,width", [(1, 1), (5, 3), (700, 1), (901, 33), (1300, 259), (700, 2051), (450, 4099), (3, 20003)])
@pytest.mark.parametrize("rd,ad", PAIRS)
def test_block_norm_odd_addresses(ops, n, width, rd, ad):
    """Contiguous arrays at addresses that only their type aligns, each another one, between NaN:
    nothing around an array, and nothing of another row, gets into a row."""
    def at(offset, t):
        flat = torch.full((t.numel() + 32,), float("nan"), dtype=t.dtype, device="cuda")
        flat[offset:offset + t.numel()] = t.reshape(-1)
        return flat[offset:offset + t.numel()].view(t.shape)

    res, x, post, pre, gate = _norm_inputs((1, n, width), rd, ad, "channel")
    dh, dy = _randn(25, 1, n, width, scale=0.5, dtype=rd), _randn(26, 1, n, width, scale=0.5, dtype=ad)
    res, x, dh, dy, post, pre, gate = (at(i, t) for i, t in zip((1, 3, 5, 7, 1, 2, 5), (res, x, dh, dy, post, pre, gate)))
    h, y = ops.block_norm(res, x, post, pre, gate, 0.35)
    want_h, want_y = P.block_norm(res, x, post, pre, gate, 0.35, 1e-6)
    P.check(h, *want_h, rd, "h")
    P.check(y, *want_y, ad, "y")
    for a in ((res, x, dh, dy, post, pre, gate), (res, x, dh, None, post, pre, gate), (res, None, None, dy, None, pre, None)):
        want = P.block_norm_grad(*a, 0.35, 1e-6)
        like = (rd, rd if a[1] is None else ad, F32, F32, gate.dtype)
        if a[1] is None and ad != rd:
            continue
        for i, g in enumerate(ops.block_norm_grad(*a, 0.35)):
            if g is not None:
                P.check(g, *want[i], like[i], str(i))
    if n > 600:
        dh[0, n // 2, -1], dy[0, n // 3, width // 2:] = float("inf"), float("nan")
        got = ops.block_norm_grad(res, x, dh, dy, post, pre, gate, 0.35)
        bad = torch.zeros(n, dtype=torch.bool, device="cuda")
        bad[n // 2] = bad[n // 3] = True
        for g in got[:2]:
            assert torch.isfinite(g[0, ~bad]).all() and not torch.isfinite(g[0, bad]).all(1).any()


def test_block_norm_empty_and_extreme(ops):
    res, x, post, pre, gate = _norm_inputs((3, 0, 16), BF16, BF16, "sample")
    h, y = ops.block_norm(res, x, post, pre, gate)
    assert h.shape == y.shape == (3, 0, 16)
    got = ops.block_norm_grad(res, x, res, x, post, pre, gate)
    assert all(not g.any() for g in got) and got[4].shape == (3, 1, 16)
    # a row of zeros has the norm 1 / sqrt(eps), a large one must not overflow its float32 sum
    res, x, post, pre, gate = _norm_inputs((2, 4, 48), F32, F32, "channel")
    res[0, 1], x[0, 1] = 0, 0
    x[0, 2], res[0, 2] = 1e15, 1e15
    x[1, 0] = 1e-30
    _check_norm(ops, res, x, post, pre, gate)
    _check_norm_grad(ops, res, x, post, pre, gate)
    # NaN and infinities stay in their rows, but for the sums over rows
    x[1, 1, 5], res[1, 2, 7] = float("nan"), float("inf")
    h, y = ops.block_norm(res, x, post, pre, gate)
    d = ops.block_norm_grad(res, x, res, x, post, pre, gate)
    good = torch.ones(2, 4, dtype=torch.bool, device="cuda")
    good[1, 1] = good[1, 2] = False
    for t in (h, y, d[0], d[1]):
        assert torch.isfinite(t[good]).all() and not torch.isfinite(t[~good]).all()
    assert torch.isnan(y[1, 1]).all()


def test_block_norm_beyond_32_bit_offsets(ops):
    n, d, last = 530001, 4104, 3  # 2.17e9 elements
    make = lambda seed: _randn(seed, last, d, dtype=BF16)  # noqa: E731
    res, x = torch.zeros(n, d, dtype=BF16, device="cuda"), torch.zeros(n, d, dtype=BF16, device="cuda")
    res[-last:], x[-last:] = make(120), make(121)
    post, pre, gate = 1 + _randn(122, d, scale=0.3), 1 + _randn(123, d, scale=0.3), _randn(124, d)
    h, y = ops.block_norm(res, x, post, pre, gate, 0.5)
    want_h, want_y = P.block_norm(make(120), make(121), post, pre, gate, 0.5, 1e-6)
    P.check(h[-last:], *want_h, BF16, "h")
    P.check(y[-last:], *want_y, BF16, "y")
    assert not h[:-last].any() and not y[:-last].any()
    del h, y
    dh, dy = torch.zeros(n, d, dtype=BF16, device="cuda"), torch.zeros(n, d, dtype=BF16, device="cuda")
    dh[-last:], dy[-last:] = make(125), make(126)
    got = ops.block_norm_grad(res, x, dh, dy, post, pre, gate, 0.5)
    want = P.block_norm_grad(make(120), make(121), make(125), make(126), post, pre, gate, 0.5, 1e-6)
    for i, like in enumerate((BF16, BF16, F32, F32, F32)):  # rows of zeros add nothing to the sums
        P.check(got[i][-last:] if i < 2 else got[i], *want[i], like, str(i))
    assert not got[0][:-last].any() and not got[1][:-last].any()


# -------------------------------------------------------------------------- distillation

def _distill_inputs(n, vocab, k, dtype, seed=30, td=F32, ids_dtype=torch.int64):
    logits = _randn(seed, n, vocab, scale=3.0, dtype=dtype)
    teacher = _randn(seed + 1, n, k, scale=3.0, dtype=td)
    ids = _tokens(seed + 2, (n, k), vocab, ids_dtype)
    weight = _randn(seed + 3, n)
    weight[n // 2] = 0
    return logits, ids, teacher, weight


def _check_distill(ops, logits, ids, teacher, weight, tau):
    v = logits.shape[-1]
    (loss, lb), (grad, gb) = P.distill(logits.reshape(-1, v), ids.reshape(-1, ids.shape[-1]),
                                       teacher.reshape(-1, ids.shape[-1]),
                                       None if weight is None else weight.reshape(-1), tau)
    got = ops.distill_loss(logits, ids, teacher, weight, tau)
    P.check(got.reshape(-1), loss, lb, F32, "loss")
    l2, g2 = ops.distill_grad(logits, ids, teacher, weight, tau)
    P.check(l2.reshape(-1), loss, lb, F32, "loss with gradient")
    P.check(g2.reshape(-1, v), grad, gb, logits.dtype, "gradient")
    l3, g3 = ops.distill_grad(logits, ids, teacher, weight, tau)
    same = lambda a, b: torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))  # noqa: E731
    assert same(l2, l3) and same(g2, g3)
    if logits.is_contiguous():
        inplace = logits.clone()
        l4, g4 = ops.distill_grad(inplace, ids, teacher, weight, tau, inplace=True)
        assert g4 is inplace and same(l4, l2) and same(g4, g2)


@pytest.mark.parametrize("n,vocab,k", [(0, 9, 3), (1, 1, 1), (1, 32000, 32), (3, 7, 5), (5, 1000, 64), (9, 1003, 17),
                                       (2, 32768, 8), (4, 65537, 100), (3, 128259, 20), (2, 300007, 33), (33, 513, 1024),
                                       (700, 260, 3), (1, 1200001, 5)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_distill(ops, n, vocab, k, dtype):
    if n == 0:
        z = torch.zeros(0, vocab, dtype=dtype, device="cuda")
        loss, grad = ops.distill_grad(z, torch.zeros(0, k, dtype=torch.int64, device="cuda"),
                                      torch.zeros(0, k, device="cuda"))
        assert loss.shape == (0,) and grad.shape == (0, vocab)
        return
    a = _distill_inputs(n, vocab, k, dtype)
    _check_distill(ops, *a, 1.0)
    _check_distill(ops, *a[:3], None, 2.5)


@pytest.mark.parametrize("td,idt", [(F32, torch.int32), (BF16, torch.int64), (F16, torch.int32)])
def test_distill_teacher_types_and_shapes(ops, td, idt):
    logits, ids, teacher, weight = _distill_inputs(12, 777, 9, BF16, td=td, ids_dtype=idt)
    _check_distill(ops, logits.reshape(3, 4, 777), ids.reshape(3, 4, 9), teacher.reshape(3, 4, 9), weight.reshape(3, 4),
                   0.5)
    _check_distill(ops, logits[0], ids[0], teacher[0], weight[0], 0.5)
    none = torch.zeros(12, 0, dtype=idt, device="cuda")
    loss, grad = ops.distill_grad(logits, none, none.to(td))
    assert not loss.any() and not grad.any()


def test_distill_strides(ops):
    wide, ids, teacher, weight = _distill_inputs(6, 520, 7, BF16)
    for z in (wide[:, :512], wide[:, 8:520], wide[:, 1:512], wide[:, 3:11], wide[::2], wide[:3].transpose(0, 1)[:3]):
        n, v = z.shape
        i = ids[:n] % v
        _check_distill(ops, z, i, teacher[:n], weight[:n], 2.0)
    both = torch.stack([ids, ids], 2)[..., 0], torch.stack([teacher, teacher], 2)[..., 1]
    _check_distill(ops, wide, *both, torch.stack([weight, weight], 1)[:, 0], 2.0)


def test_distill_repeated_ids(ops):
    logits, ids, teacher, weight = _distill_inputs(8, 50, 40, F32)
    ids[0] = 7                    # one id forty times
    ids[1] = ids[1] % 2
    _check_distill(ops, logits, ids, teacher, weight, 1.0)


def test_distill_masks(ops):
    """Lists that are short or empty, masked vocabularies, masked rows that hold anything."""
    inf = float("inf")
    for dtype in (F32, F16, BF16):
        logits, ids, teacher, weight = _distill_inputs(12, 4099, 6, dtype)
        weight[:] = 0.5
        ids[0, 2:] = -1                       # a short list
        ids[1] = -1                           # no list
        ids[2] = torch.tensor([4099, 2**40, -2**40, -1, 5000, 2**31], device="cuda")
        teacher[3, :5] = -inf                 # one valid entry: p = 1
        teacher[4] = -inf
        logits[5, 100:] = -inf                # a masked vocabulary, the teacher's ids within it
        ids[5] = torch.arange(6, device="cuda") * 3
        logits[6] = -inf                      # nothing left: q = 0, the loss infinite
        weight[7], logits[7], teacher[7] = 0, float("nan"), float("nan")
        weight[8], logits[8] = 0, inf
        logits[9, 17], logits[10, 5] = float("nan"), inf
        logits[11] = torch.finfo(dtype).min   # the type's lowest value everywhere: uniform
        if dtype is F32:
            logits[11] = -1e30
        _check_distill(ops, logits, ids, teacher, weight, 1.0)
        loss, grad = ops.distill_grad(logits, ids, teacher, weight)
        for r in (1, 2, 4, 7, 8):
            assert not grad[r].any() and float(loss[r]) == 0
        assert float(loss[6]) == inf and torch.isnan(grad[9]).all() and torch.isnan(loss[10])
        # the student gives a teacher's entry no chance
        logits, ids, teacher, weight = _distill_inputs(2, 300, 3, dtype)
        logits[0, ids[0, 1]] = -inf
        weight[:] = 1
        _check_distill(ops, logits, ids, teacher, weight, 1.0)


def test_distill_far_logits(ops):
    """Maxima far from zero and wide spreads: exponentials relative to the maximum."""
    logits, ids, teacher, weight = _distill_inputs(4, 3001, 8, F32)
    logits[0] += 1e4
    logits[1] -= 3e4
    logits[2] *= 100
    teacher[3] += 500
    _check_distill(ops, logits, ids, teacher, weight, 1.0)
    _check_distill(ops, logits, ids, teacher, weight, 30.0)


@pytest.mark.parametrize("vocab", [3001, 32000, 128259])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distill_uneven_rows(ops, vocab, dtype):
    """A logit far above all others, or all of them far below, at the end of a row; beginnings
    that are masked; every one of them in every part of the row."""
    inf = float("inf")
    logits, ids, teacher, weight = _distill_inputs(9, vocab, 6, dtype)
    weight[:] = 1
    logits[0, -1] = 300
    logits[1, vocab // 2] = 88
    logits[2, :vocab - 5] = -inf
    ids[2] = torch.arange(6, device="cuda") + vocab - 6
    logits[3, :vocab - 5] = torch.finfo(dtype).min
    logits[4, :vocab // 2] = -inf
    logits[4, vocab // 2:] -= 100
    logits[5, vocab // 3:] = -200
    logits[6, vocab // 2:] += 200
    logits[7] = -1e4
    logits[8] = 0
    _check_distill(ops, logits, ids, teacher, weight, 1.0)


def test_distill_long_lists_of_one_id(ops):
    logits, ids, teacher, weight = _distill_inputs(3, 5000, 1024, F32)
    ids[0] = 4999
    ids[1] = torch.arange(1024, device="cuda") % 3
    ids[2, ::2] = -1
    _check_distill(ops, logits, ids, teacher, weight, 2.0)


def test_calls_at_once_on_two_streams(ops):
    """Calls that overlap on the GPU share nothing."""
    t = [_chain_inputs(s) for s in (110, 130)]
    want = [_chain(ops, x) for x in t]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for x, s in zip(t, streams):
            with torch.cuda.stream(s):
                outs.append(_chain(ops, x))
    torch.cuda.synchronize()
    for i, (loss, grads) in enumerate(outs):
        assert torch.equal(loss, want[i % 2][0])
        assert all(torch.equal(grads[k], want[i % 2][1][k]) for k in grads)


def test_distill_rows_beyond_32_bit_offsets(ops):
    n, vocab = 17000, 128256  # 2.18e9 elements
    logits = torch.zeros(n, vocab, dtype=BF16, device="cuda")
    logits[-2:] = _randn(40, 2, vocab, scale=2.0, dtype=BF16)
    ids, teacher = _tokens(41, (n, 4), vocab), _randn(42, n, 4)
    weight = torch.zeros(n, device="cuda")
    weight[-2:] = 3.0
    loss, grad = ops.distill_grad(logits, ids, teacher, weight, 1.0, inplace=True)
    fresh = _randn(40, 2, vocab, scale=2.0, dtype=BF16)
    (want, lb), (g, gb) = P.distill(fresh, ids[-2:], teacher[-2:], weight[-2:], 1.0)
    P.check(loss[-2:], want, lb, F32)
    P.check(grad[-2:], g, gb, BF16)
    assert not grad[:-2].any()


# ---------------------------------------------------------------- streams, graphs, together

def _chain(ops, t):
    """Lookup, two blocks (a product each), logits, loss and the whole way back, as a
    training step that leaves the gradients of its parameters; returns loss and gradients."""
    e = ops.embedding_gather(t["table"], t["tokens"], 8.0, dtype=BF16)
    h0, y0 = ops.block_norm(e, pre_weight=t["pre0"])
    x1 = y0 @ t["w1"]
    h1, y1 = ops.block_norm(h0, x1, t["post1"], t["pre1"], t["gate"], 0.5)
    logits = y1 @ t["head"]
    loss, dz = ops.distill_grad(logits, t["ids"], t["teacher"], t["weight"], 2.0, inplace=True)
    d_y1 = dz @ t["head"].t()
    d_h0, d_x1, d_post1, d_pre1, d_gate = ops.block_norm_grad(h1, x1, None, d_y1, t["post1"], t["pre1"], t["gate"], 0.5)
    d_y0 = d_x1 @ t["w1"].t()
    d_e, _, _, d_pre0, _ = ops.block_norm_grad(h0, None, d_h0, d_y0, None, t["pre0"])
    d_table = ops.embedding_grad(d_e, t["tokens"], t["table"].shape[0], 8.0, dtype=F32)
    d_w1 = y0.reshape(-1, 128).t() @ d_x1.reshape(-1, 128)
    d_head = y1.reshape(-1, 128).t() @ dz.reshape(-1, t["head"].shape[1])
    return loss, dict(table=d_table, w1=d_w1, head=d_head, post1=d_post1, pre0=d_pre0, pre1=d_pre1, gate=d_gate)


def _chain_inputs(seed):
    b, s, d, v, k = 2, 37, 128, 1003, 9
    return dict(table=_randn(seed, v, d, scale=0.1), tokens=_tokens(seed + 1, (b, s), v),
                w1=_randn(seed + 2, d, d, scale=0.09, dtype=BF16), head=_randn(seed + 3, d, v, scale=0.09, dtype=BF16),
                post1=1 + _randn(seed + 4, d, scale=0.1), pre0=1 + _randn(seed + 5, d, scale=0.1),
                pre1=1 + _randn(seed + 6, d, scale=0.1), gate=_randn(seed + 7, d, scale=0.5),
                ids=_tokens(seed + 8, (b, s, k), v), teacher=_randn(seed + 9, b, s, k, scale=2.0),
                weight=torch.full((b, s), 1 / (b * s), device="cuda"))


def test_chain_gradients_against_autograd_in_float64(ops):
    t = _chain_inputs(50)
    loss, grads = _chain(ops, t)
    p = {k: v.double().requires_grad_() if v.is_floating_point() else v for k, v in t.items()}
    e = p["table"][p["tokens"]] * 8.0
    (_, _), (y0, _) = P.block_norm(e, None, None, p["pre0"], None, 1.0, 1e-6)
    (_, _), (y1, _) = P.block_norm(e, y0 @ p["w1"], p["post1"], p["pre1"], p["gate"], 0.5, 1e-6)
    z = (y1 @ p["head"]).reshape(-1, 1003)
    (want, _), _ = P.distill(z, t["ids"].reshape(-1, 9), t["teacher"].reshape(-1, 9), t["weight"].reshape(-1), 2.0)
    names = list(grads)
    exact = torch.autograd.grad(want.sum(), [p[k] for k in names])
    # about ten 16-bit roundings of half a step (2^-9 of the value for bfloat16 twice over) lie on the
    # way to each gradient; in the 2-norm they add up like independent errors, below 16 * 2^-8 in any case
    assert float((loss.double().reshape(-1) - want.detach()).norm() / want.detach().norm()) < 16 * 2.0 ** -8
    for name, g in zip(names, exact):
        rel = float((grads[name].double() - g).norm() / g.norm())
        assert rel < 16 * 2.0 ** -8, (name, rel)


def test_inside_autograd_functions(ops):
    """As the forward and backward of torch.autograd.Function: gradients against autograd's of the
    formulas in float64."""
    class Embedding(torch.autograd.Function):
        @staticmethod
        def forward(ctx, weight, tokens, scale):
            ctx.save_for_backward(tokens)
            ctx.rows, ctx.scale, ctx.dtype = weight.shape[0], scale, weight.dtype
            return ops.embedding_gather(weight, tokens, scale)

        @staticmethod
        def backward(ctx, grad):
            return ops.embedding_grad(grad, ctx.saved_tensors[0], ctx.rows, ctx.scale, dtype=ctx.dtype), None, None

    class Norm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, residual, x, post, pre):
            h, y = ops.block_norm(residual, x, post, pre, None, 0.5)
            ctx.save_for_backward(h, x, post, pre)
            return h, y

        @staticmethod
        def backward(ctx, d_h, d_y):
            h, x, post, pre = ctx.saved_tensors
            d_residual, d_x, d_post, d_pre, _ = ops.block_norm_grad(h, x, d_h, d_y, post, pre, None, 0.5)
            return d_residual, d_x, d_post, d_pre

    class Distill(torch.autograd.Function):
        @staticmethod
        def forward(ctx, logits, ids, teacher):
            loss, grad = ops.distill_grad(logits, ids, teacher)
            ctx.save_for_backward(grad)
            return loss

        @staticmethod
        def backward(ctx, d_loss):
            return ctx.saved_tensors[0] * d_loss[:, None], None, None

    v, d, n = 301, 64, 23
    table, other = _randn(150, v, d, scale=0.3), _randn(151, n, d)
    post, pre = 1 + _randn(152, d, scale=0.2), 1 + _randn(153, d, scale=0.2)
    tok, ids, teacher = _tokens(154, n, v), _tokens(155, (n, 4), v), _randn(156, n, 4)
    leaves = [t.clone().requires_grad_() for t in (table, other, post, pre)]
    e = Embedding.apply(leaves[0], tok, 2.0)
    h, y = Norm.apply(leaves[1], e, leaves[2], leaves[3])
    z = (h + y) @ table.t()
    Distill.apply(z, ids, teacher).sum().backward()
    wide = [t.double().requires_grad_() for t in (table, other, post, pre)]
    (h, _), (y, _) = P.block_norm(wide[1], wide[0][tok] * 2.0, wide[2], wide[3], None, 0.5, 1e-6)
    P.distill((h + y) @ table.double().t(), ids, teacher, None, 1.0)[0][0].sum().backward()
    # float32 throughout: a few hundred roundings of 2^-24 on the way to a gradient
    for got, want in zip(leaves, wide):
        assert float((got.grad.double() - want.grad).norm() / want.grad.norm()) < 1000 * 2.0 ** -24


def test_chain_feeds_the_optimizer(ops):
    """The gradients go to CRESSO5.step() as they are."""
    import cresso_b200
    from oracle import cresso5_oracle as O
    t = _chain_inputs(60)
    names = ("table", "post1", "pre0", "pre1", "gate")
    kw = dict(rank=8, hash_bins=64, hash_tables=2)
    params = [torch.nn.Parameter(t[k].clone()) for k in names]
    mirror = [torch.nn.Parameter(t[k].cpu().clone()) for k in names]
    opt, ref = cresso_b200.CRESSO5(params, **kw), O.OracleCRESSO5(mirror, **kw)
    for _ in range(2):
        with torch.no_grad():
            _, grads = _chain(ops, {**t, **dict(zip(names, params))})
        for p, m, k in zip(params, mirror, names):
            p.grad = grads[k].to(p.dtype)
            m.grad = p.grad.cpu()
        opt.step()
        ref.step()
    for p, m in zip(params, mirror):
        d = (p.detach().cpu().double() - m.detach().double()).pow(2).mean().sqrt()
        assert float(d / m.detach().double().pow(2).mean().sqrt()) <= 1e-5  # the step's own parameter tolerance


def test_other_stream_and_graphs(ops):
    """On a stream of their own, and captured: two graphs replayed in turn with new inputs
    give what eager calls give, bit for bit."""
    t = [_chain_inputs(70), _chain_inputs(90)]
    want = [_chain(ops, x) for x in t]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss, grads = _chain(ops, t[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(loss, want[0][0]) and all(torch.equal(grads[k], want[0][1][k]) for k in grads)
    static = [{k: v.clone() for k, v in x.items()} for x in t]
    graphs, outs = [], []
    for x in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_chain(ops, x))
        graphs.append(g)
    for order in ((0, 1), (1, 0)):
        for i, g in enumerate(graphs):
            for k, v in static[i].items():
                v.copy_(t[order[i]][k])
        for g in graphs + graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            loss, grads = want[order[i]]
            assert torch.equal(outs[i][0], loss) and all(torch.equal(outs[i][1][k], grads[k]) for k in grads)


def test_library_counts_the_launches(ops):
    from cresso_b200 import _lib
    before = _lib.launch_count()
    w = _randn(80, 8, 8)
    ops.embedding_gather(w, _tokens(81, 3, 8))
    assert _lib.launch_count() > before
