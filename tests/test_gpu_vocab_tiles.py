"""The large tiles of the vocabulary operators (256 x 256) over several slices of the summed index, whole and half last columns
of tiles, and the gradient of the bias reduced a piece of the vocabulary at a time: against the formula in float64, with the
tolerances derived in test_gpu_vocab.py and, for vocabularies whose log-likelihoods are a logarithm of their size, the
logarithm's own steps (4 U |LSE|, derived in fuzz_vocab.py).  float32 operands are two fp16 limbs, good to 2^-22."""
import ctypes
import math

import pytest
import torch

from test_gpu_vocab import DT, U, close, oracle

pytestmark = pytest.mark.gpu


def bias_share(T, V, H, dt, bias_dt=torch.float32):
    """Bytes of the backward's workspace that the gradient of the bias adds."""
    from lvae import _native as N
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
    three, out, got = ctypes.c_int64 * 3, ctypes.c_int64(0), []
    q = N.VocabProblem(256, 256, 256, 256, three(1, 1, T), three(0, 0, H), three(0, 0, 1), V, H, -100, H, code[dt], code[bias_dt], 0)
    for want_bias in (0, 1):
        N.check(N.lib().lvae_vocab_ll_bwd_workspace_bytes(q, 1, 1, want_bias, out))
        got.append(out.value)
    return got[1] - got[0]


def up(n, to):
    return -(-n // to) * to


# tokens, how many count (last columns of 44, 129, 128, 256, 1, 130, 100 and 64 tokens), words, width (2, 3, 4, 4, 12, 13, 5
# and 1 slices of 64)
SHAPES = [(300, 300, 17000, 128), (512, 385, 17000, 192), (512, 384, 17001, 200), (400, 256, 20000, 256), (700, 513, 12000, 768),
          (700, 130, 12001, 831), (600, 100, 12000, 320), (832, 832, 9000, 64)]


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,kept,V,H", SHAPES)
def test_large_tiles(dt, T, kept, V, H):
    from lvae import decoder_ops as D
    # a wave's column sums of the bias gradient: 4 for 256 tokens of the large tiles, 8 of the small ones
    assert bias_share(T, V, H, DT[dt]) == up(T, 256) // 256 * 4 * up(V, 256) * 4, "another tile than the test is for"
    g = torch.Generator(device="cuda").manual_seed(T + V)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    h = r(T, H).to(DT[dt])
    w = (r(V, H + 8) * (2.0 / math.sqrt(H))).to(DT[dt])[:, :H]          # rows a pitch apart
    b = r(V)
    y = torch.randint(0, V, (T,), device="cuda", generator=g)
    y[torch.randperm(T, device="cuda", generator=g)[kept:]] = -100
    y[(y != -100).nonzero()[0]] = V - 1
    gy = r(T)
    o = oracle(h, w, b, y, gy)
    ts = [h.clone().requires_grad_(), w.detach().requires_grad_(), b.clone().requires_grad_()]
    ll = D.token_log_likelihood(ts[0], ts[1], y, ts[2])
    ll.backward(-gy)
    log_steps = 4 * U * torch.maximum(o["lse"].abs(), o["ll"].abs())
    close(ll, o["ll"].cpu(), (o["tol"] + log_steps).cpu(), "ll")
    close(ts[0].grad, o["dh"].cpu(), o["tol_dh"].cpu(), "d_hidden")
    close(ts[1].grad, o["dw"].cpu(), o["tol_dw"].cpu(), "d_weight")
    close(ts[2].grad, o["db"].cpu(), o["tol_db"].cpu(), "d_bias")
    assert (ts[0].grad[y == -100] == 0).all()


@pytest.mark.parametrize("dt,bias_dt", [("bf16", "f32"), ("bf16", "bf16"), ("f32", "f16")])
def test_bias_gradient_a_piece_at_a_time(dt, bias_dt):
    """So many tokens and words that the column sums of all pieces would pass 256 MiB: those of one piece exist at a time."""
    from lvae import decoder_ops as D
    T, V, H = 66000, 65200, 16
    assert bias_share(T, V, H, DT[dt], DT[bias_dt]) < up(T, 256) // 256 * 4 * up(V, 256) * 4 // 4, "all pieces at once"
    g = torch.Generator(device="cuda").manual_seed(0)
    h = torch.randn(T, H, device="cuda", generator=g).to(DT[dt])
    w = (torch.randn(V, H, device="cuda", generator=g) / 4).to(DT[dt])
    b = torch.zeros(V, device="cuda", dtype=DT[bias_dt], requires_grad=True)
    y = torch.randint(0, V, (T,), device="cuda", generator=g)
    D.vocab_cross_entropy(h, w, y, b, reduction="sum").backward()
    mass = torch.zeros(V, device="cuda", dtype=torch.float64)
    for rows in range(0, T, 2000):
        mass += torch.softmax(h[rows:rows + 2000].double() @ w.double().t(), 1).sum(0)
    count = torch.bincount(y, minlength=V)
    want = mass - count
    # a logit is off by tol: S below 40, |h| < 5, |w| < 1.3, 16 terms of mean 0.16.  A column sum adds up 16 lanes of 4 column
    # tiles, 64 values, in float32, the rest in float64; rounded to the type of the bias at the end
    tol = 2 * (H + 16) * 2 * U * 40 + 2.0 ** -20 + 8 * U * 11
    bound = mass * (2 * tol + 2.0 ** -21) + 64 * U * (mass + count) + want.abs() * (torch.finfo(DT[bias_dt]).eps / 2 + U)
    assert ((b.grad.double() - want).abs() <= bound).all()


def test_sequences_in_float16():
    """Gradient of whole sentences whose samples share their words, more tokens than one decoding step has."""
    from lvae import decoder_ops as D
    B, K, L, H, V = 3, 4, 11, 72, 400
    g = torch.Generator().manual_seed(3)
    h = torch.randn(B, K, L, H, generator=g).half()
    w = (torch.randn(V, H, generator=g) / 8).half()
    y = torch.randint(0, V, (B, L), generator=g)
    y[0, 7:] = -100
    y[2] = -100
    gs = torch.randn(B, K, generator=g)
    flat = y[:, None].expand(B, K, L).reshape(-1)
    o = oracle(h.reshape(-1, H), w, None, flat, gs[..., None].expand(B, K, L).reshape(-1))
    hc, wc = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    out = D.sequence_log_likelihood(hc, wc, y.cuda()[:, None])
    want = o["ll"].view(B, K, L).sum(-1)
    close(out, want, o["tol"].view(B, K, L).sum(-1) + U * want.abs(), "log p(x|z)")
    out.backward(-gs.cuda())
    close(hc.grad, o["dh"].view(B, K, L, H), o["tol_dh"].view(B, K, L, H), "d_hidden")
    close(wc.grad, o["dw"], o["tol_dw"], "d_weight")


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,V,H", [(20, 300, 64), (150, 500, 72), (2100, 300, 64), (700, 12000, 128)])
def test_each_gradient_alone(dt, T, V, H):
    """A frozen decoder, or frozen hidden states: what is asked for has the bits that it has beside the others."""
    from lvae import decoder_ops as D
    g = torch.Generator(device="cuda").manual_seed(T)
    data = [torch.randn(T, H, device="cuda", generator=g).to(DT[dt]), (torch.randn(V, H, device="cuda", generator=g) / 8).to(DT[dt]),
            torch.randn(V, device="cuda", generator=g)]
    y = torch.randint(0, V, (T,), device="cuda", generator=g)
    y[::7] = -100

    def gradients(wanted):
        ts = [t.clone().requires_grad_(k in wanted) for k, t in enumerate(data)]
        return torch.autograd.grad(D.vocab_cross_entropy(ts[0], ts[1], y, ts[2]), [ts[k] for k in wanted])
    whole = gradients((0, 1, 2))
    for wanted in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
        for k, got in zip(wanted, gradients(wanted)):
            assert torch.equal(got, whole[k]), wanted
