"""Vocabulary operators (lvae.decoder_ops) at the limits that the C header states."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_most_words(dt):
    """2^26 - 1 words whose rows are copied for the tiles: 2^22 times 16 rows, more than one launch of 2^32 threads holds
    one workgroup each for.  The last word is a target too.

    Tolerances.  A logit is one product, exact in float32 or good to 2^-22, plus the bias: |l| < 2^4, off by 2^-18 at most.
    The sum over the words joins 2^18 / 16 partial sums one after the other, each addition and rescaling within 2U, and 300
    terms besides: relative (2^14 + 300) 2U = 2^-8.9.  A gradient of a hidden state is sum_v p_v w_v with |w| <= 1, and
    the mass of p is off by as much: 2^-8 together, the rounding of G and of the result included (bf16: 2^-8 each)."""
    from lvae import decoder_ops as D
    V, T = (1 << 26) - 1, 65
    g = torch.Generator(device="cuda").manual_seed(0)
    w = (2 * torch.rand(V, 1, device="cuda", generator=g) - 1).to(torch.float32 if dt == "f32" else torch.bfloat16)
    h = (2 * torch.rand(T, 1, device="cuda", generator=g) - 1).to(w.dtype)
    y = torch.randint(0, V, (T,), device="cuda", generator=g)
    y[0], y[1], y[2] = V - 1, V - 1000000, 0
    # words beyond the 16 (2^22 - 2^16) rows that the copies of one launch held at most weigh 20 times the others
    b = torch.zeros(V, device="cuda")
    b[-(1 << 20):] = 3.0
    hr = h.clone().requires_grad_()
    ll = D.token_log_likelihood(hr, w, y, b)
    ll.sum().backward()
    wd = w.double()[:, 0]
    for t in range(T):
        l = wd * h[t, 0].double() + b
        lse = torch.logsumexp(l, 0)
        assert abs((l[y[t]] - lse).item() - ll[t].item()) <= 2.0 ** -8, t
        want = wd[y[t]] - (torch.exp(l - lse) * wd).sum()
        assert abs(want.item() - hr.grad[t, 0].item()) <= 2.0 ** -8 + (0 if dt == "f32" else 3 * 2.0 ** -8), t


@pytest.mark.parametrize("n,length", [((1 << 26) - 1, 1), ((1 << 25) + 5, 3), (1000, 70), (3, 0)])
def test_most_segments(n, length):
    """2^26 - 1 sums: one workgroup for four of them would be 2^32 threads.  float64 inside, rounded once."""
    from lvae import _native as N
    x = torch.randn(n, length, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n))
    out = torch.full((n + 4,), 7.0, device="cuda")
    N.check(N.lib().lvae_segment_sum_f32(x.data_ptr(), n, length, out.data_ptr(), N.raw_stream(0)))
    want = x.double().sum(1)
    assert ((out[:n].double() - want).abs() <= U * want.abs() + length * 2.0 ** -48).all()
    assert (out[n:] == 7).all()
