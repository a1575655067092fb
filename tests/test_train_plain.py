"""The float64 formulas that the training operators are held to: their gradients
agree with automatic differentiation and with central differences of the forward
formulas, on the CPU."""

import torch

import _train_plain as P


def _leaf(gen, *shape):
    return torch.randn(shape, generator=gen, dtype=torch.float64).requires_grad_()


def test_embedding_grad_is_the_lookups_gradient():
    gen = torch.Generator().manual_seed(1)
    tokens = torch.tensor([[3, 5, 3], [9, 4, -1]])
    w = torch.randn(4, 3, generator=gen, dtype=torch.float64)
    g = torch.randn(2, 3, 3, generator=gen, dtype=torch.float64)

    def total(w):
        return float((P.gather(w, tokens, 0.7, 3, torch.float32)[0] * g).sum())

    value, _ = P.embedding_grad(g, tokens, 4, 0.7, 3)
    for r in range(4):
        for c in range(3):
            step = torch.zeros_like(w)
            step[r, c] = 1e-4
            assert abs((total(w + step) - total(w - step)) / 2e-4 - float(value[r, c])) < 1e-8
    masked, _ = P.embedding_grad(g, tokens, 4, 0.7, 3, padding=3)
    assert torch.equal(masked[0], torch.zeros(3, dtype=torch.float64)) and torch.equal(masked[1:], value[1:])


def test_block_norm_grad_is_the_forwards_gradient():
    gen = torch.Generator().manual_seed(2)
    shape, eps, scale = (2, 3, 5), 1e-3, 0.6
    for post_on in (True, False):
        for gate_shape in (None, (5,), (2, 1, 5), (2, 3, 5)):
            res, x, pre = _leaf(gen, *shape), _leaf(gen, *shape), _leaf(gen, 5)
            post = _leaf(gen, 5) if post_on else None
            gate = None if gate_shape is None else _leaf(gen, *gate_shape)
            dh, dy = _leaf(gen, *shape).detach(), _leaf(gen, *shape).detach()

            def f(*leaves):
                it = iter(leaves)
                r, xx, pr = next(it), next(it), next(it)
                po = next(it) if post_on else None
                ga = next(it) if gate is not None else None
                (h, _), (y, _) = P.block_norm(r, xx, po, pr, ga, scale, eps)
                return h, y

            leaves = [t for t in (res, x, pre, post, gate) if t is not None]
            assert torch.autograd.gradcheck(f, leaves)  # central differences
            h, y = f(*leaves)
            want = iter(torch.autograd.grad([h, y], leaves, [dh, dy]))
            got = P.block_norm_grad(h.detach(), x.detach(), dh, dy, None if post is None else post.detach(),
                                    pre.detach(), None if gate is None else gate.detach(), scale, eps)
            for k, on in ((0, True), (1, True), (3, True), (2, post_on), (4, gate is not None)):
                assert (got[k] is not None) == on
                if on:
                    torch.testing.assert_close(got[k][0], next(want), rtol=1e-10, atol=1e-12)


def test_distill_gradient_is_the_losses_gradient():
    gen = torch.Generator().manual_seed(3)
    z = _leaf(gen, 4, 7)
    ids = torch.tensor([[0, 3, 3], [6, -1, 2], [-1, 9, -1], [1, 2, 5]])
    teacher = torch.randn(4, 3, generator=gen)
    teacher[3, 1] = -torch.inf
    weight = torch.tensor([0.5, 2.0, 1.0, -0.25])

    def f(z):
        return P.distill(z, ids, teacher, weight, 1.5)[0][0].sum()

    assert torch.autograd.gradcheck(f, (z,))
    torch.testing.assert_close(P.distill(z.detach(), ids, teacher, weight, 1.5)[1][0], torch.autograd.grad(f(z), z)[0],
                               rtol=1e-10, atol=1e-12)


def test_distill_loss_is_the_divergence():
    """With the whole vocabulary as the teacher's list it is the divergence of the two softmaxes."""
    gen = torch.Generator().manual_seed(4)
    z, u = torch.randn(3, 9, generator=gen), torch.randn(3, 9, generator=gen)
    loss = P.distill(z, torch.arange(9).expand(3, 9), u, None, 2.0)[0][0]
    p, q = torch.softmax(u.double() / 2, 1), torch.softmax(z.double() / 2, 1)
    torch.testing.assert_close(loss, 4 * (p * (p.log() - q.log())).sum(1))
