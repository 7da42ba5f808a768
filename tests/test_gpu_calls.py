"""Calls of the vocabulary and gradient operators that a kernel reading plain memory would answer wrongly."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


def test_forward_mode_derivatives_are_refused():
    from lvae import _native as N, decoder_ops as D, grad_ops as G
    h, w, b = torch.randn(3, 8, device="cuda"), torch.randn(5, 8, device="cuda"), torch.randn(5, device="cuda")
    y = torch.zeros(3, dtype=torch.int64, device="cuda")
    t, out = torch.ones(6, device="cuda"), torch.zeros(6, device="cuda")
    with fwd.dual_level():
        with pytest.raises(N.LvaeError, match="hidden carries a tangent"):
            D.token_log_likelihood(fwd.make_dual(h, h), w, y, b)
        with pytest.raises(N.LvaeError, match=r"grads\[0\] carries a tangent"):
            G.clip_grads([fwd.make_dual(t, t)], 1.0)
        with pytest.raises(N.LvaeError, match=r"out\[0\] carries a tangent"):
            G.clip_grads([t], 1.0, out=[fwd.make_dual(out, out)])
        # forward over backward
        hr = h.clone().requires_grad_()
        ll = D.token_log_likelihood(hr, w, y, b)
        one = torch.ones_like(ll)
        with pytest.raises(N.LvaeError, match="upstream gradient carries a tangent"):
            torch.autograd.grad(ll, hr, fwd.make_dual(one, one), retain_graph=True)
        plain, = torch.autograd.grad(ll, hr, one)          # tensors without a tangent are served as ever
        assert torch.isfinite(plain).all()
    assert (t == 1).all() and (out == 0).all()


def test_negated_views():
    """The imaginary part of a conjugate is a view whose memory holds the other sign; nothing else shows it."""
    from lvae import decoder_ops as D, grad_ops as G
    for T in (9, 100):
        g = torch.Generator(device="cuda").manual_seed(T)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)
        h, w, b = r(T, 8), r(300, 8), r(300)
        y = torch.randint(0, 300, (T,), device="cuda", generator=g)

        def step(h, w, b):
            ll = D.token_log_likelihood(h, w, y, b)
            return [ll.detach()] + list(torch.autograd.grad(ll.sum(), (h, w, b)))
        negated = [torch._neg_view(-t) for t in (h, w, b)]
        assert all(t.is_neg() and torch.equal(t, u) for t, u in zip(negated, (h, w, b)))
        want = step(*[t.requires_grad_() for t in (h, w, b)])
        for a, e in zip(step(*[t.requires_grad_() for t in negated]), want):
            assert torch.equal(a, e)
        one = torch.complex(h.detach()[:, 0], h.detach()[:, 1]).conj().imag[:, None]       # a single column, two apart
        w1 = w.detach()[:, :1].contiguous()
        assert one.is_neg() and torch.equal(D.token_log_likelihood(one, w1, y), D.token_log_likelihood((-h.detach()[:, 1:2]).contiguous(), w1, y))
    t = torch.randn(50, device="cuda")
    for src, dst in ((torch._neg_view(t.clone()), torch.empty(50, device="cuda")), ((-t), torch._neg_view(torch.empty(50, device="cuda"))),
                     (torch._neg_view(t.clone()), torch._neg_view(torch.empty(50, device="cuda")))):
        G.clip_grads([src], 0.5, out=[dst])
        want = torch.empty(50, device="cuda")
        G.clip_grads([-t], 0.5, out=[want])
        assert torch.equal(dst, want)
    n = torch._neg_view(t.clone())
    G.clip_grads([n], 0.5)
    assert torch.equal(n, want)


def test_a_refused_clip_changes_nothing():
    """Neither values nor version counters: a graph that has saved one of the tensors still runs backward."""
    from lvae import _native as N, grad_ops as G
    t, u = torch.full((100,), 2.0, device="cuda"), torch.full((100,), 3.0, device="cuda")
    wants = torch.full((100,), 2.0, device="cuda", requires_grad=True)
    x = torch.ones(100, device="cuda", requires_grad=True)
    out = x * t
    for call, error in ((lambda: G.clip_grads([t, t], 1.0), "share memory"), (lambda: G.clip_grads([t[:60], t[50:]], 1.0), "share memory"),
                        (lambda: G.clip_grads([u, u.clone()], 1.0, out=[t, t]), "share memory"),
                        (lambda: G.clip_grads([t, wants], 1.0), "requires grad"), (lambda: G.clip_grads([u, u], 1.0, out=[t, wants]), "requires grad")):
        before = t._version, u._version, wants._version
        with pytest.raises(N.LvaeError, match=error):
            call()
        assert (t._version, u._version, wants._version) == before
        assert (t == 2).all() and (u == 3).all() and (wants == 2).all()
    out.sum().backward()
    assert torch.equal(x.grad, t)
    out = x * t
    before = u._version
    G.clip_grads([u], 1.0, out=[t])
    assert u._version == before
    with pytest.raises(RuntimeError, match="inplace"):            # what was written is noticed as before
        out.sum().backward()
    column = torch.ones(30, 4, device="cuda")
    out = x[:30, None] * column
    G.clip_grads([column[:, 1]], 0.5)                            # through a dense copy
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


def test_the_factor_of_clipping_is_rounded_once():
    """n ones have the norm sqrt(n): each becomes the factor itself, max_norm / (sqrt(n) + 1e-6) in float64, rounded to float32 (half
    a step, 2^-24 of the value; 2^-40 of it for the float64 arithmetic)."""
    from lvae import grad_ops as G
    for n in range(2, 400, 7):
        for bound in (0.1, 1.0 / 3.0, 0.7):
            want = bound / (n ** 0.5 + 1e-6)
            t = [torch.ones(n, device="cuda")]
            G.clip_grads(t, bound)
            assert (t[0].double() - want).abs().max().item() <= (2.0 ** -24 + 2.0 ** -40) * want, (n, bound)
        t = [torch.ones(n, device="cuda")]
        G.clip_grads(t, 0.1, norm_type=float("inf"))
        assert (t[0].double() - 0.1 / (1 + 1e-6)).abs().max().item() <= (2.0 ** -24 + 2.0 ** -40) * 0.1
    # a norm beyond float32, which reads as inf, of elements that are not: they are scaled by what it is
    t = [torch.full((100,), 3e38, device="cuda")]
    assert G.clip_grads(t, 1e10).item() == float("inf")
    assert (t[0].double() - 1e9).abs().max().item() <= (2.0 ** -23 + 2.0 ** -40) * 1e9        # the factor and the product
