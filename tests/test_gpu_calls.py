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
