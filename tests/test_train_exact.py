"""The training operators on inputs that show a single element left out of a sum, taken twice
or put elsewhere: whole numbers, whose float32 sums are exact, and rows with one large element
at every position of a short row and around every place where a long one is cut."""

import pytest
import torch

import _train_plain as P

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from cresso_b200 import ops as _ops
    return _ops


def _gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


# ---------------------------------------------------------------------------- embedding

def _whole_numbers(seed, *shape, dtype):
    return torch.randint(-8, 9, shape, generator=_gen(seed), device="cuda").to(dtype)


# positions and widths around the sizes at which the tiles of positions change, each width with another access
@gpu
@pytest.mark.parametrize("n,width", [(4000, 8), (4096, 5), (4097, 6), (131072, 8), (131072, 12), (131072, 6), (131072, 5),
                                     (131072, 128), (131072, 129), (131073, 16), (140000, 12), (140000, 6), (140000, 7),
                                     (70000, 264), (1048576, 8), (1048577, 8), (1048577, 12), (1048577, 6), (1048577, 3)])
@pytest.mark.parametrize("gd,od", [(BF16, F32), (F32, F32), (F16, BF16)])
def test_embedding_grad_of_whole_numbers(ops, n, width, gd, od):
    """Sums below 2^24 of whole numbers are exact in any order: the result is the only one possible."""
    rows = 61
    g = _whole_numbers(1, n, width, dtype=gd)
    tok = (torch.rand(n, generator=_gen(2), device="cuda", dtype=torch.float64) ** 3 * rows).long()
    tok[n // 3:n // 2] = 7       # a long run of one row
    tok[::11] = -1
    inside = tok >= 0
    total = torch.zeros(rows, width, dtype=torch.int64, device="cuda")
    total.index_add_(0, tok[inside], g[inside].long())
    assert torch.equal(ops.embedding_grad(g, tok, rows, 0.25, dtype=od), (total.double() * 0.25).to(od))
    into = _whole_numbers(3, rows + 5, width, dtype=od)  # the last rows have no token
    want = into.double()
    want[:rows] += total.double() * 0.25
    ops.embedding_grad(g, tok, rows + 5, 0.25, into=into)
    assert torch.equal(into, want.to(od))


@gpu
@pytest.mark.parametrize("width", [1, 3, 6, 12, 64, 264, 2050])
@pytest.mark.parametrize("wd,od", [(BF16, F32), (F32, BF16), (F16, F16)])
def test_gather_of_whole_numbers(ops, width, wd, od):
    w = _whole_numbers(4, 301, width, dtype=wd)
    tok = torch.randint(-3, 330, (2003,), generator=_gen(5), device="cuda")
    want = torch.where(((tok >= 0) & (tok < 301))[:, None], w[tok.clamp(0, 300)].double() * 0.5, 0.0)
    assert torch.equal(ops.embedding_gather(w, tok, 0.5, dtype=od), want.to(od))


# ---------------------------------------------------------------------------- rows with one large element

def _places(width, every):
    """All positions of a short row; of a long one its ends, the surroundings of its halves, quarters and
    eighths, and some in between."""
    if width <= every:
        return torch.arange(width)
    near = torch.arange(-25, 25)
    at = [torch.arange(33), width - 1 - torch.arange(33), torch.randint(width, (64,), generator=_gen(9, "cpu"))]
    at += [width * k // 8 + near for k in range(1, 8)]
    return torch.unique(torch.cat(at).clamp(0, width - 1))


def _hot(places, width, value, dtype, device="cuda"):
    t = torch.zeros(len(places), width, dtype=dtype, device=device)
    t[torch.arange(len(places)), places] = value
    return t


def _offset(t, k):
    """The same contiguous tensor k elements behind an aligned address."""
    flat = torch.empty(t.numel() + k, dtype=t.dtype, device=t.device)
    flat[k:] = t.reshape(-1)
    return flat[k:].view(t.shape)


@gpu
@pytest.mark.parametrize("width", [1, 7, 33, 130, 511, 513, 520, 1030, 1031, 2050, 2051, 2560, 4096, 4099, 4104, 8192, 8193,
                                   8200, 16385, 16392, 20001, 32776, 40000, 65535, 65536])
@pytest.mark.parametrize("rd,ad", [(F32, F32), (F32, BF16), (F16, F16)])
@pytest.mark.parametrize("gate_on", [None, "channel", "full"])
def test_norms_of_rows_with_one_large_element(ops, width, rd, ad, gate_on):
    """Without its large element in one of the sums, h, y, d_residual or d_x of the row is another one by far;
    the sums over the rows have one row's share in each column."""
    at = _places(width, 1100)
    n = len(at)
    x, res = _hot(at, width, 2.0, ad), _hot(at, width, -1.0, rd)
    post, pre = (1 + 0.2 * torch.randn(width, generator=_gen(s), device="cuda") for s in (1, 2))
    gate = None
    if gate_on is not None:
        gate = (1.5 + 0.2 * torch.randn(*((n, width) if gate_on == "full" else (width,)), generator=_gen(3),
                                        device="cuda").clamp(-2, 2)).to(ad)
    for shift in (0, 1):
        r, xx = _offset(res, shift), _offset(x, shift)
        h, y = ops.block_norm(r, xx, post, pre, gate, 0.5)
        want_h, want_y = P.block_norm(res, x, post, pre, gate, 0.5, 1e-6)
        P.check(h, *want_h, rd, "h")
        P.check(y, *want_y, ad, "y")
        hh, dh, dy = _offset(_hot(at, width, 1.0, rd), shift), _hot(at, width, 1.0, rd), _hot(at, width, 1 / 64, ad)
        got = ops.block_norm_grad(hh, xx, dh, dy, post, pre, gate, 0.5)
        want = P.block_norm_grad(hh, xx, dh, dy, post, pre, gate, 0.5, 1e-6)
        for name, g, w, t in zip(("d_residual", "d_x", "d_post", "d_pre", "d_gate"), got, want,
                                 (rd, ad, post.dtype, pre.dtype, ad)):
            if g is not None:
                P.check(g, *w, t, name)


@gpu
@pytest.mark.parametrize("vocab,rows_at_once", [(5, None), (67, None), (1003, None), (2053, 8), (4099, None), (16411, 8),
                                                (32768, None), (32771, 3), (65537, None), (128259, None), (128264, 8),
                                                (300007, None)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_distill_of_rows_with_one_large_logit(ops, vocab, rows_at_once, dtype):
    """A row's sum is its large logit: without it, or with it twice, the loss and the gradient there are
    others by far.  Few rows at once are cut into more parts."""
    at = _places(vocab, 4099)
    logits = _hot(at, vocab, 20.0, dtype)
    ids = ((at + 1 + torch.arange(len(at)) % max(1, vocab - 1)) % vocab)[:, None].cuda()  # another place than the large logit's
    teacher = torch.zeros(len(at), 1, device="cuda")
    step = rows_at_once or len(at)
    for i in range(0, len(at), step):
        z, d, u = logits[i:i + step], ids[i:i + step], teacher[i:i + step]
        (loss, lb), (grad, gb) = P.distill(z, d, u, None, 1.0)
        P.check(ops.distill_loss(z, d, u), loss, lb, F32, "loss")
        got_loss, got = ops.distill_grad(z, d, u)
        P.check(got_loss, loss, lb, F32, "loss with gradient")
        P.check(got, grad, gb, dtype, "gradient")


# ------------------------------------------------------------------ that these inputs show it (no GPU)

@pytest.mark.parametrize("vocab", [1003, 20011])
def test_a_word_left_out_of_a_long_row_is_seen(vocab):
    at = _places(vocab, 64)
    logits = _hot(at, vocab, 20.0, F32, "cpu")
    ids, teacher = ((at + 1) % vocab)[:, None], torch.zeros(len(at), 1)
    (loss, lb), (grad, gb) = P.distill(logits, ids, teacher, None, 1.0)
    P.check(loss.float(), loss, lb, F32)
    for k, j in list(enumerate(at.tolist()))[::7]:
        damaged = logits[k:k + 1].clone()
        damaged[0, j] = -torch.inf
        (bad, _), _ = P.distill(damaged, ids[k:k + 1], teacher[k:k + 1], None, 1.0)
        with pytest.raises(AssertionError):
            P.check(bad.float(), loss[k:k + 1], lb[k:k + 1], F32)


@pytest.mark.parametrize("width", [513, 20001, 65536])
def test_a_column_left_out_of_a_norm_is_seen(width):
    at = _places(width, 64)[::9]
    x, res, w = _hot(at, width, 2.0, F32, "cpu"), _hot(at, width, -1.0, F32, "cpu"), torch.ones(width)
    (h, hb), (y, yb) = P.block_norm(res, x, w, w, None, 0.5, 1e-6)
    k = torch.arange(len(at))
    for row, j in zip(k.tolist(), at.tolist()):
        # x's element missing in the first mean, h's in the second one, each with the others in place
        bad_h = h[row].clone()
        bad_h[j] = -1.0 + 0.5 * 2.0 / (1e-6 ** 0.5)
        with pytest.raises(AssertionError):
            P.check(bad_h.float(), h[row], hb[row], F32)
        bad_y = y[row].clone()
        bad_y[j] = h[row, j] / (1e-6 ** 0.5)
        with pytest.raises(AssertionError):
            P.check(bad_y.float(), y[row], yb[row], F32)
