"""Token and sequence log-likelihoods, cross entropy over the vocabulary and their gradients (lvae.decoder_ops) against
the formula in float64.

Tolerances.  u = 2^-24 is half a step of float32, e = finfo(type).eps / 2 half a step of the operand type.
 * A logit is a sum of H products that are exact in float32 (16-bit operands) or good to 2^-22 (three bf16 limbs, the
   products below 2^-24 left out), added in float32: off by at most a = (H + 16) 2u S, S = max_v sum_h |h||w|.
 * The LSE takes over that error, an exponential and a logarithm (2^-21 together, relative to terms of at most 1, i.e.
   absolute in the logarithm) and two roundings at the size of the logits: tol = 2 a + 2^-20 + 8 u max|l|.
 * A softmax value p is then good to p (2 tol + 2^-21); G = (p - onehot) g is rounded once to the operand type (e |G|; fp16
   also to multiples of 2^-38 of the largest upstream gradient, its subnormals after scaling; half of that is added).
 * A gradient adds up V or T such values in float32: sum |dG||w| + (n + 16) 2u sum |G||w|, and is rounded once, e |d|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def inputs(T, V, H, dt, seed=0, bias=True, ignore=0.2, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(T, H, generator=g).to(dt)
    w = (torch.randn(V, H, generator=g) * scale / math.sqrt(H)).to(dt)
    b = torch.randn(V, generator=g).to(dt) if bias else None
    y = torch.randint(0, V, (T,), generator=g)
    y[torch.rand(T, generator=g) < ignore] = -100
    return h, w, b, y


def oracle(h, w, b, y, gy=None, ignore=-100):
    """ll, tolerances and gradients in float64, for [T, H] hidden states of 16 or 32 bits."""
    dt = h.dtype
    e = torch.finfo(dt).eps / 2
    hd, wd = h.double(), w.double()
    keep = y != ignore
    hd = torch.where(keep[:, None], hd, 0.0)
    l = hd @ wd.T + (0.0 if b is None else b.double())
    lse = torch.logsumexp(l, 1)
    at = y.clamp(min=0)
    ll = torch.where(keep, l.gather(1, at[:, None])[:, 0] - lse, 0.0)
    H, V, T = h.shape[1], w.shape[0], h.shape[0]
    S = (hd.abs() @ wd.abs().T).amax(1)
    fin = torch.where(torch.isfinite(l), l, 0.0)
    tol = 2 * (H + 16) * 2 * U * S + 2.0 ** -20 + 8 * U * fin.abs().amax(1)
    out = {"ll": ll, "tol": torch.where(keep, tol, 0.0), "lse": lse}
    if gy is None:
        return out
    gy = torch.where(keep, gy.double(), 0.0)
    p = torch.exp(l - lse[:, None])
    G = p.clone()
    G[torch.arange(T), at] -= 1.0
    G = G * gy[:, None]
    dG = G.abs() * (e if dt != torch.float32 else 2 * U) + p * gy.abs()[:, None] * (2 * tol[:, None] + 2.0 ** -21) + 2 * U * gy.abs()[:, None]
    if dt == torch.float16:
        dG = dG + 2.0 ** -39 * gy.abs().max()
    dG = torch.where(keep[:, None], dG, 0.0)
    n = keep.sum().item()
    out["dh"] = G @ wd
    out["tol_dh"] = dG @ wd.abs() + (V + 16) * 2 * U * (G.abs() @ wd.abs()) + e * out["dh"].abs()
    out["dw"] = G.T @ hd
    out["tol_dw"] = dG.T @ hd.abs() + (n + 16) * 2 * U * (G.abs().T @ hd.abs()) + e * out["dw"].abs()
    out["db"] = G.sum(0)
    e_b = 0.0 if b is None else torch.finfo(b.dtype).eps / 2
    out["tol_db"] = (p * gy.abs()[:, None] * (2 * tol[:, None] + 2.0 ** -21)).sum(0) + (n + 16) * 2 * U * G.abs().sum(0) + e_b * out["db"].abs()
    tiny = torch.finfo(dt).smallest_normal * e * 2      # the last step of the result's subnormals
    for k in ("tol_dh", "tol_dw"):
        out[k] = out[k] + tiny
    if b is not None:
        out["tol_db"] = out["tol_db"] + torch.finfo(b.dtype).smallest_normal * e_b * 2
    return out


def close(got, want, tol, what):
    got = got.detach().double().cpu().reshape(want.shape)
    bad = ~((got - want).abs() <= tol) & ~(got == want)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / tol).nan_to_num(nan=math.inf).max():.3g} tol"


SHAPES = [(1, 1, 1), (1, 17, 5), (3, 64, 64), (16, 999, 331), (17, 130, 72), (64, 1000, 128), (65, 257, 64), (100, 513, 100),
          (129, 700, 192), (256, 256, 256), (257, 1029, 320), (300, 2000, 33)]


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,V,H", SHAPES)
def test_forward(dt, T, V, H):
    from lvae import decoder_ops as D
    h, w, b, y = inputs(T, V, H, DT[dt], seed=T + V, bias=T % 2 == 0)
    o = oracle(h, w, b, y)
    ll = D.token_log_likelihood(h.cuda(), w.cuda(), y.cuda(), bias=None if b is None else b.cuda())
    assert ll.dtype == torch.float32 and ll.shape == (T,)
    close(ll, o["ll"], o["tol"], "ll")


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,V,H", SHAPES)
def test_gradients(dt, T, V, H):
    from lvae import decoder_ops as D
    h, w, b, y = inputs(T, V, H, DT[dt], seed=T + V, bias=T % 2 == 0)
    gy = torch.randn(T, generator=torch.Generator().manual_seed(1))
    o = oracle(h, w, b, y, gy)
    hc, wc = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    bc = None if b is None else b.cuda().requires_grad_()
    ll = D.token_log_likelihood(hc, wc, y.cuda(), bias=bc)
    close(ll, o["ll"], o["tol"], "ll")
    # d ll: the oracle's G is that of -ll
    ll.backward(-gy.cuda())
    close(hc.grad, o["dh"], o["tol_dh"], "d_hidden")
    close(wc.grad, o["dw"], o["tol_dw"], "d_weight")
    assert hc.grad.dtype == h.dtype and wc.grad.dtype == w.dtype
    if b is not None:
        close(bc.grad, o["db"], o["tol_db"], "d_bias")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_many_pieces_and_splits(dt):
    """A vocabulary of several pieces, and few output tiles over long sums (split products)."""
    from lvae import decoder_ops as D
    for T, V, H in ((150, 40000, 64), (2100, 300, 64)):
        h, w, b, y = inputs(T, V, H, DT[dt], seed=5)
        gy = torch.rand(T, generator=torch.Generator().manual_seed(1)) + 0.5
        o = oracle(h, w, b, y, gy)
        hc, wc, bc = h.cuda().requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()
        D.token_log_likelihood(hc, wc, y.cuda(), bias=bc).backward(-gy.cuda())
        close(hc.grad, o["dh"], o["tol_dh"], "d_hidden")
        close(wc.grad, o["dw"], o["tol_dw"], "d_weight")
        close(bc.grad, o["db"], o["tol_db"], "d_bias")


@pytest.mark.parametrize("T", [5, 300])
def test_padding_may_hold_anything(T):
    from lvae import decoder_ops as D
    h, w, b, y = inputs(T, 600, 64, torch.bfloat16, ignore=0.5)
    o = oracle(h, w, b, y, torch.ones(T))
    bad = h.clone()
    bad[y == -100] = float("nan")
    bad[(y == -100) & (torch.arange(T) % 2 == 0)] = float("inf")
    hc, wc, bc = bad.cuda().requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()
    ll = D.token_log_likelihood(hc, wc, y.cuda(), bias=bc)
    close(ll, o["ll"], o["tol"], "ll")
    (-ll.sum()).backward()
    close(hc.grad, o["dh"], o["tol_dh"], "d_hidden")
    close(wc.grad, o["dw"], o["tol_dw"], "d_weight")
    close(bc.grad, o["db"], o["tol_db"], "d_bias")
    assert (hc.grad[(y == -100).cuda()] == 0).all()


@pytest.mark.parametrize("T", [4, 200])
def test_no_token_counts(T):
    from lvae import decoder_ops as D
    h, w, b, y = inputs(T, 300, 64, torch.bfloat16)
    y[:] = -100
    hc, wc, bc = h.cuda().requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()
    loss = D.vocab_cross_entropy(hc, wc, y.cuda(), bias=bc)
    loss.backward()
    assert loss.item() == 0.0
    for g in (hc.grad, wc.grad, bc.grad):
        assert (g == 0).all()


@pytest.mark.parametrize("T", [7, 130])
@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min])
def test_banned_words(T, low):
    """A bias of -inf, or of the lowest value, takes words out; a banned target is -inf (or the lowest value) likely."""
    from lvae import decoder_ops as D
    h, w, _, y = inputs(T, 500, 64, torch.bfloat16, ignore=0.0)
    b = torch.zeros(500)
    b[::3] = low
    y = torch.where(y % 3 == 0, (y + 1) % 500, y)
    y = torch.where(y % 3 == 0, 1, y)
    o = oracle(h, w, b, y, torch.ones(T))
    hc, wc, bc = h.cuda().requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()
    ll = D.token_log_likelihood(hc, wc, y.cuda(), bias=bc)
    tol = 2 * (64 + 16) * 2 * U * (h.double().abs() @ w.double().abs().T).amax(1) + 2.0 ** -20 + 8 * U * 30
    close(ll, o["ll"], tol, "ll")
    (-ll.sum()).backward()
    assert (wc.grad[::3] == 0).all() and (bc.grad[::3] == 0).all()
    assert torch.isfinite(hc.grad).all()
    y[0] = 0
    ll = D.token_log_likelihood(h.cuda(), w.cuda(), y.cuda(), bias=b.cuda())
    assert ll[0].item() == -math.inf or ll[0].item() <= -3e38
    # nothing is left: not a number, as 0 / 0
    b[:] = -math.inf
    assert torch.isnan(D.token_log_likelihood(h.cuda(), w.cuda(), y.cuda(), bias=b.cuda())).all()


@pytest.mark.parametrize("T", [7, 130])
@pytest.mark.parametrize("bad", [-1, 500, 2 ** 40, -2 ** 62])
def test_target_outside_the_vocabulary(T, bad):
    from lvae import decoder_ops as D
    h, w, b, y = inputs(T, 500, 64, torch.bfloat16)
    y[2] = bad
    o = oracle(h, w, b, torch.where(y == bad, -100, y))
    hc = h.cuda().requires_grad_()
    ll = D.token_log_likelihood(hc, w.cuda(), y.cuda(), bias=b.cuda())
    assert torch.isnan(ll[2])
    rest = torch.arange(T) != 2
    close(ll[rest.cuda()], o["ll"][rest], o["tol"][rest], "ll")
    ll.sum().backward()
    assert torch.isnan(hc.grad[2]).all() and torch.isfinite(hc.grad[rest.cuda()]).all()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("B,K,L", [(2, 3, 1), (3, 5, 17), (1, 1, 4)])
def test_sequences(dt, B, K, L):
    """Targets shared by the samples of a sentence, hidden states cut out of longer ones, a sentence of padding."""
    from lvae import decoder_ops as D
    H, V = 72, 400
    g = torch.Generator().manual_seed(3)
    full = torch.randn(B, K, L + 2, H, generator=g).to(DT[dt])
    h = full[:, :, 1:-1]
    w = (torch.randn(V, H, generator=g) / 8).to(DT[dt])
    y = torch.randint(0, V, (B, L + 3), generator=g)
    y[B - 1] = -7
    yc = y.cuda()[:, 2:-1]
    o = oracle(h.reshape(-1, H), w, None, y[:, None, 2:-1].expand(B, K, L).reshape(-1), torch.ones(B * K * L), ignore=-7)
    fc, wc = full.cuda().requires_grad_(), w.cuda().requires_grad_()
    out = D.sequence_log_likelihood(fc[:, :, 1:-1], wc, yc[:, None], ignore_index=-7)
    assert out.shape == (B, K)
    want = o["ll"].view(B, K, L).sum(-1)
    close(out, want, o["tol"].view(B, K, L).sum(-1) + U * want.abs(), "log p(x|z)")
    assert (out[B - 1] == 0).all()
    gs = torch.randn(B, K, generator=g)
    o = oracle(h.reshape(-1, H), w, None, y[:, None, 2:-1].expand(B, K, L).reshape(-1), gs[..., None].expand(B, K, L).reshape(-1), ignore=-7)
    out.backward(-gs.cuda())
    close(fc.grad[:, :, 1:-1].reshape(-1, H), o["dh"], o["tol_dh"], "d_hidden")
    assert (fc.grad[:, :, 0] == 0).all() and (fc.grad[:, :, -1] == 0).all()
    close(wc.grad, o["dw"], o["tol_dw"], "d_weight")


def test_reductions():
    from lvae import decoder_ops as D
    h, w, b, y = (t.cuda() for t in inputs(90, 300, 64, torch.float32))
    none = D.vocab_cross_entropy(h, w, y, b, reduction="none")
    n = int((y != -100).sum())
    s, m = D.vocab_cross_entropy(h, w, y, b, reduction="sum"), D.vocab_cross_entropy(h, w, y, b)
    want = none.double().sum().item()
    assert abs(s.item() - want) <= 2 * U * abs(want) and abs(m.item() - want / n) <= 2 * U * abs(want / n)
    for red, factor in (("sum", 1.0), ("mean", 1.0 / n)):
        hc = h.clone().requires_grad_()
        (3 * D.vocab_cross_entropy(hc, w, y, b, reduction=red)).backward()
        o = oracle(h.cpu(), w.cpu(), b.cpu(), y.cpu(), torch.full((90,), 3 * factor))
        close(hc.grad, o["dh"], o["tol_dh"], red)


def test_gradient_against_differences():
    """Central differences of the sum along random directions, float32.  The sum is about 700 and off by 700 * 2^-22 at
    each end: 700 * 2^-22 / eps = 0.006 at eps = 0.03; the third derivative along a unit direction is below 1 a token
    that it moves (|h| ~ 1, softmax moments), eps^2 / 6 * 120 < 0.02."""
    from lvae import decoder_ops as D
    h, w, b, y = (t.cuda() for t in inputs(150, 300, 64, torch.float32))
    f = lambda h, w, b: D.vocab_cross_entropy(h, w, y, b, reduction="sum")
    ts = [t.clone().requires_grad_() for t in (h, w, b)]
    grads = torch.autograd.grad(f(*ts), ts)
    g = torch.Generator(device="cuda").manual_seed(2)
    for k in range(3):
        d = torch.randn(ts[k].shape, device="cuda", generator=g)
        d /= d.norm()
        eps = 0.03
        up, down = [t.detach() for t in ts], [t.detach() for t in ts]
        up[k], down[k] = up[k] + eps * d, down[k] - eps * d
        num = (f(*up).double() - f(*down).double()).item() / (2 * eps)
        assert abs(num - (grads[k].double() * d.double()).sum().item()) < 0.026


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_layouts(dt):
    """Rows off 16-byte boundaries, row pitches, transposed and broadcast operands give what dense ones give."""
    from lvae import decoder_ops as D
    for T, V, H in ((9, 200, 64), (140, 200, 64)):
        h, w, b, y = (t.cuda() for t in inputs(T, V, H, DT[dt]))
        want = D.token_log_likelihood(h, w, y, b)
        off = torch.zeros(T * H + 1, device="cuda", dtype=h.dtype)[1:].view(T, H)
        off.copy_(h)
        wide = torch.full((V, H + 3), float("nan"), device="cuda", dtype=w.dtype)
        wide[:, :H] = w
        bb = torch.stack([b, b], 1)[:, 0]
        o = oracle(h.cpu(), w.cpu(), b.cpu(), y.cpu())
        for hh, ww in ((off, w), (h, wide[:, :H]), (h.t().contiguous().t(), w), (h, w.t().contiguous().t())):
            close(D.token_log_likelihood(hh, ww, y, bb), o["ll"], o["tol"], "ll")
        one = h[:1].expand(T, H)
        o = oracle(one.cpu(), w.cpu(), b.cpu(), y.cpu())
        close(D.token_log_likelihood(one, w, y, b), o["ll"], o["tol"], "ll of one row for all")
        assert torch.isfinite(want).all()
        hp, wp = off.detach().requires_grad_(), wide[:, :H].detach().requires_grad_()
        D.token_log_likelihood(hp, wp, y, b).sum().backward()
        o = oracle(h.cpu(), w.cpu(), b.cpu(), y.cpu(), -torch.ones(T))
        close(hp.grad, o["dh"], o["tol_dh"], "d_hidden")
        close(wp.grad, o["dw"], o["tol_dw"], "d_weight")
    # four token axes that do not join
    h = torch.randn(3, 4, 5, 6, 64, device="cuda").to(DT[dt]).permute(3, 0, 2, 1, 4)
    y = torch.randint(0, V, h.shape[:-1], device="cuda")
    o = oracle(h.reshape(-1, 64).cpu(), w.cpu(), b.cpu(), y.reshape(-1).cpu())
    close(D.token_log_likelihood(h, w, y, b).reshape(-1), o["ll"], o["tol"], "ll")


def test_same_bits_every_time_and_on_another_stream():
    from lvae import decoder_ops as D
    h, w, b, y = (t.cuda() for t in inputs(700, 3000, 128, torch.bfloat16))

    def step():
        ts = [t.detach().requires_grad_() for t in (h, w, b)]
        loss = D.vocab_cross_entropy(ts[0], ts[1], y, ts[2])
        return [loss.detach()] + list(torch.autograd.grad(loss, ts))
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    third = step()
    torch.cuda.synchronize()
    for a, b2, c in zip(first, second, third):
        assert torch.equal(a, b2) and torch.equal(a, c)


@pytest.mark.parametrize("T", [8, 200])
def test_captured_and_replayed(T):
    from lvae import decoder_ops as D
    h, w, b, y = (t.cuda() for t in inputs(T, 900, 64, torch.bfloat16))

    def step(h, w, b, y):
        ts = [t.detach().requires_grad_() for t in (h, w, b)]
        loss = D.vocab_cross_entropy(ts[0], ts[1], y, ts[2])
        return [loss.detach()] + list(torch.autograd.grad(loss, ts))
    sh, sy = h.clone(), y.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(sh, w, b, sy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sh, w, b, sy)
    for k in range(4):
        h2, _, _, y2 = (t.cuda() for t in inputs(T, 900, 64, torch.bfloat16, seed=10 + k, ignore=0.3 * k))
        sh.copy_(h2)
        sy.copy_(y2)
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(out, step(h2, w, b, y2)):
            assert torch.equal(a, e)


def test_training_step_of_the_text_model():
    """The operators together, as a step uses them: encode tail, log p(x|z), the importance-weighted bound, backward,
    norm of all gradients and clipping."""
    from lvae import decoder_ops as D, encoder_ops, estimators, grad_ops
    B, K, L, H, V, Z = 6, 4, 9, 64, 500, 32
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    mu, lv = r(B, Z).requires_grad_(), (0.1 * r(B, Z)).requires_grad_()
    up = (r(Z, H) / 8).requires_grad_()
    words, bias = (r(V, H) / 8).requires_grad_(), r(V).requires_grad_()
    eps, prior, pos = r(B, K, Z), r(B, Z), r(L, H)
    y = torch.randint(0, V, (B, L), device="cuda", generator=g)
    y[1, 4:] = -100

    def forward(ll_of):
        tail = encoder_ops.encode_tail(mu, lv, n_samples=K, eps=eps, prior_sample=prior)
        states = (tail["latent_z"] @ up)[:, :, None] + pos
        log_p_x_z = ll_of(states)
        return (log_p_x_z + tail["log_p_z"] - tail["log_q_z_x"]), tail, log_p_x_z
    params = [mu, lv, up, words, bias]
    logw, tail, lp = forward(lambda s: D.sequence_log_likelihood(s, words, y[:, None], bias=bias))
    loss = -(torch.logsumexp(logw, 1) - math.log(K)).mean()
    loss.backward()
    got = [p.grad.clone() for p in params]
    for p in params:
        p.grad = None

    def plain(s):
        lg = torch.log_softmax(s.double() @ words.double().t() + bias.double(), -1)
        t = y[:, None].expand(B, K, L)
        return torch.where(t != -100, lg.gather(-1, t.clamp(min=0)[..., None])[..., 0], 0.0).sum(-1)
    logw2, _, lp2 = forward(plain)
    (-(torch.logsumexp(logw2, 1) - math.log(K)).mean()).backward()
    # float32 throughout on both sides but for the plain logits: 2^-24 * (a few hundred additions) of sums of order 10
    assert (lp.double() - lp2.double()).abs().max() < 2e-4
    for a, p in zip(got, params):
        assert (a - p.grad).norm() <= 2e-5 * p.grad.norm()
    iw = estimators.iw_log_p_x(lp.detach(), tail["log_p_z"].detach(), tail["log_q_z_x"].detach())
    assert abs(iw.mean().item() + loss.item()) < 1e-4
    want = math.sqrt(sum(p.grad.double().square().sum().item() for p in params))
    before = [p.grad.clone() for p in params]
    norm = grad_ops.clip_grad_norm_(params, want / 2)
    assert abs(norm.item() - want) <= 4 * U * want
    for p, q in zip(params, before):
        assert torch.allclose(p.grad, q * 0.5, rtol=1e-6, atol=0)


def test_bias_gradient_piece_by_piece():
    """So many tokens and words that the bias gradient's column sums are reduced after every piece of the vocabulary."""
    from lvae import decoder_ops as D
    T, V, H = 66000, 65000, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    h = torch.randn(T, H, device="cuda", generator=g).bfloat16()
    w = (torch.randn(V, H, device="cuda", generator=g) / 4).bfloat16()
    b = torch.zeros(V, device="cuda", requires_grad=True)
    y = torch.randint(0, V, (T,), device="cuda", generator=g)
    D.vocab_cross_entropy(h, w, y, b, reduction="sum").backward()
    want, mass = torch.zeros(V, device="cuda", dtype=torch.float64), torch.zeros(V, device="cuda", dtype=torch.float64)
    for rows in range(0, T, 2000):
        p = torch.softmax(h[rows:rows + 2000].double() @ w.double().t(), 1)
        mass += p.sum(0)
    want = mass - torch.bincount(y, minlength=V)
    tol = 2 * (H + 16) * 2 * U * 40 + 2.0 ** -20 + 8 * U * 10      # of a logit; S below 40: |h| < 5, |w| < 1.3, 16 terms of mean 0.16
    bound = mass * (2 * tol + 2.0 ** -21) + 64 * U * (mass + torch.bincount(y, minlength=V)) + U * want.abs()
    assert ((b.grad.double() - want).abs() <= bound).all()


def test_float32_beside_much_larger_values():
    """float32 operands are scaled by one power of two a tensor: rows far below the largest element keep their bits.  Word 0
    holds 2^20 where the hidden states are 0, the others are 2^-10 small, 2^-30 of it: below what one fp16 limb holds
    without subnormals.  Their logits are sums of 63 products of 2^-10 and 1, good to 2^-22 each and 2^-51 * 2^20 absolute."""
    from lvae import decoder_ops as D
    T, V, H = 100, 40, 64
    g = torch.Generator().manual_seed(9)
    h = torch.randn(T, H, generator=g)
    h[:, 0] = 0.0
    w = torch.randn(V, H, generator=g) * 2.0 ** -10
    w[0] = 0.0
    w[0, 0] = 2.0 ** 20
    y = torch.randint(0, V, (T,), generator=g)
    o = oracle(h, w, None, y, torch.ones(T))
    S = (h.double().abs() @ w.double().abs().T).amax(1)
    tol = 2 * (H * 2.0 ** -31 * 5 + (H + 16) * 2 * U * S) + 2.0 ** -20 + 8 * U * 5
    hc, wc = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    ll = D.token_log_likelihood(hc, wc, y.cuda())
    close(ll, o["ll"], tol, "ll")
    (-ll.sum()).backward()
    close(wc.grad, o["dw"], o["tol_dw"] + 2.0 ** -21 * T, "d_weight")
    # d_hidden: column 0 sums 2^20 (softmax); the others are of the small rows alone
    close(hc.grad[:, 0], o["dh"][:, 0], 2.0 ** 20 * 2.0 ** -18, "d_hidden, large")
    close(hc.grad[:, 1:], o["dh"][:, 1:], 2.0 ** -10 * (V + 5) * 5 * 2.0 ** -18, "d_hidden, small")


@pytest.mark.parametrize("T", [9, 200])
def test_wide_rows_and_unlikely_words(T):
    """Logits over a range of a few hundred: softmax values down to 0, no overflow; the gradient of words whose
    probability is about 2^-40 keeps its relative accuracy in float32 (the limbs of G have a scale each)."""
    from lvae import decoder_ops as D
    h, w, b, y = inputs(T, 300, 128, torch.float32, ignore=0.0, scale=3.0)
    b = b - 28.0 * (torch.arange(300) % 2)          # every other word e^-28 as likely
    y = y - y % 2
    o = oracle(h, w, b, y, torch.ones(T))
    hc, wc, bc = h.cuda().requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()
    ll = D.token_log_likelihood(hc, wc, y.cuda(), bias=bc)
    close(ll, o["ll"], o["tol"], "ll")
    (-ll.sum()).backward()
    rare = torch.arange(300) % 2 == 1
    p = torch.exp(h.double() @ w.double().T + b.double() - o["lse"][:, None])[:, rare]
    # p is good to 2 tol relative (2^-12 asked, the logits are of order 10 and 128 products), its limbs to 2^-22, or to
    # 2^-51 / 2^-28 of the largest |g| = 1 absolute: 2^-50
    bound = (p * 2.0 ** -12 + 2.0 ** -50).T @ h.double().abs() + (T + 16) * 2 * U * (p.T @ h.double().abs())
    close(wc.grad[rare.cuda()], o["dw"][rare], bound, "d_weight of unlikely words")
    big = b.clone()
    big[4] = 400.0                                   # one word takes everything
    o = oracle(h, w, big, y)
    ll = D.token_log_likelihood(h.cuda(), w.cuda(), y.cuda(), bias=big.cuda())
    close(ll, o["ll"], o["tol"], "ll")


def test_saved_tensors_laid_out_anew_at_the_old_address():
    """A hook of the saved tensors may hand back the hidden states with other strides where they were before."""
    from lvae import decoder_ops as D
    T, V, H = 140, 300, 64
    h, w, b, y = inputs(T, V, H, torch.float32)
    o = oracle(h, w, b, y, -torch.ones(T))
    wide = torch.zeros(T, 2 * H, device="cuda")
    wide[:, :H] = h.cuda()
    hc = wide[:, :H].detach().requires_grad_()

    def unpack(kept):
        t, dense = kept
        if t.dim() != 2 or t.stride(0) != 2 * H:
            return t
        t.as_strided((T, H), (H, 1)).copy_(dense)
        return t.as_strided((T, H), (H, 1))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (t, t.contiguous().clone()), unpack):
        ll = D.token_log_likelihood(hc, w.cuda(), y.cuda(), b.cuda())
    ll.sum().backward()
    close(hc.grad, o["dh"], o["tol_dh"], "d_hidden")


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_one_bad_upstream_gradient(dt, bad):
    """It spoils its own token's gradient; the other tokens' stay what they are, small ones too."""
    from lvae import decoder_ops as D
    T, V, H = 140, 300, 64
    h, w, b, y = inputs(T, V, H, DT[dt], ignore=0.0)
    gy = torch.randn(T, generator=torch.Generator().manual_seed(1)) * 1e-5
    gy[3] = 0.0
    o = oracle(h, w, b, y, gy)
    gy[3] = bad
    hc = h.cuda().requires_grad_()
    D.token_log_likelihood(hc, w.cuda(), y.cuda(), b.cuda()).backward(-gy.cuda())
    others = torch.arange(T) != 3
    close(hc.grad[others], o["dh"][others], o["tol_dh"][others], "d_hidden")
    assert not torch.isfinite(hc.grad[3]).any()


def test_refusals_on_the_gpu():
    from lvae import _native as N, decoder_ops as D
    h, w, y, b = torch.zeros(70, 8).cuda(), torch.zeros(5, 8).cuda(), torch.zeros(70, dtype=torch.int64).cuda(), torch.zeros(5).cuda()
    for f in (D.token_log_likelihood, D.vocab_cross_entropy):
        for hh in (h, h.clone().requires_grad_()):
            for args, error in (
                    ((hh.half(), w, y), TypeError), ((hh, w.bfloat16(), y), TypeError), ((hh.double(), w.double(), y), TypeError),
                    ((hh, w, y.int()), TypeError), ((hh, w, y, b.double()), TypeError), ((hh, w.tolist(), y), TypeError),
                    ((hh, w.to_sparse(), y), TypeError),
                    ((hh, w[:, :7], y), ValueError), ((hh, w[0], y), ValueError), ((hh[0, 0], w, y), ValueError),
                    ((hh, w, y[:69]), ValueError), ((hh, w, y[None]), ValueError), ((hh, w, y, b[:4]), ValueError),
                    ((hh, w, y, b[None]), ValueError), ((hh, w[:0], y), ValueError), ((hh[:, :0], w[:, :0], y), ValueError),
                    ((hh, w, y, b, 1 << 63), OverflowError), ((hh, w, y, b, 0.5), TypeError),
                    ((hh.cpu(), w, y), N.LvaeError), ((hh, w.cpu(), y), N.LvaeError), ((hh, w, y.cpu()), N.LvaeError),
                    ((hh, w, y, b.cpu()), N.LvaeError)):
                with pytest.raises(error):
                    f(*args)
    with pytest.raises(N.LvaeError, match="65536"):
        D.token_log_likelihood(torch.zeros(70, 65537).cuda(), torch.zeros(5, 65537).cuda(), y)


def test_with_autograd():
    """Twice through a kept graph; no second derivatives; changes in place are noticed; nothing is recorded without need."""
    from lvae import _native as N, decoder_ops as D
    for T in (20, 150):
        h, w, b, y = (t.cuda() for t in inputs(T, 300, 64, torch.float32))
        hr = h.clone().requires_grad_()
        loss = D.vocab_cross_entropy(hr, w, y, b)
        first, = torch.autograd.grad(loss, hr, retain_graph=True)
        again, = torch.autograd.grad(loss, hr, create_graph=True)
        assert torch.equal(first, again)
        with pytest.raises(N.LvaeError, match="second derivatives"):
            again.sum().backward()
        h2 = hr * 1.0
        loss = D.vocab_cross_entropy(h2, w, y, b)
        h2.mul_(2.0)
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
        with torch.no_grad():
            assert not D.token_log_likelihood(hr, w, y, b).requires_grad
        with torch.inference_mode():
            D.token_log_likelihood(hr, w, y, b)
        # a broadcast input: its gradient is the sum over the places it went to
        one = h[:1].clone().requires_grad_()
        D.vocab_cross_entropy(one.expand(T, 64), w, y, b, reduction="sum").backward()
        o = oracle(h[:1].expand(T, 64).cpu(), w.cpu(), b.cpu(), y.cpu(), torch.ones(T))
        close(one.grad, o["dh"].sum(0, keepdim=True), o["tol_dh"].sum(0, keepdim=True) + T * U * o["dh"].abs().sum(0, keepdim=True), "d_hidden")


def test_two_at_once():
    """Two streams with operators of their own under way at the same time, forward and backward."""
    from lvae import decoder_ops as D
    work = [tuple(t.cuda() for t in inputs(T, 5000, 128, torch.bfloat16, seed=T)) for T in (300, 700)]

    def step(h, w, b, y):
        ts = [t.detach().requires_grad_() for t in (h, w, b)]
        loss = D.vocab_cross_entropy(ts[0], ts[1], y, ts[2])
        return [loss.detach()] + list(torch.autograd.grad(loss, ts))
    want = [step(*x) for x in work]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(step(*work[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        for r in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[k]))


@pytest.mark.parametrize("T", [40, 150])
def test_backward_without_what_the_forward_kept(T):
    """Through the C entry points: the backward makes the limbs itself, to the same bits."""
    import ctypes
    from lvae import _native as N, decoder_ops as D
    V, H = 1000, 72
    h, w, b, y = (t.cuda() for t in inputs(T, V, H, torch.float32))
    ts = [t.clone().requires_grad_() for t in (h, w, b)]
    want = torch.autograd.grad(D.vocab_cross_entropy(ts[0], ts[1], y, ts[2], reduction="sum"), ts)
    three, lib, n = ctypes.c_int64 * 3, N.lib(), ctypes.c_int64(0)
    q = N.VocabProblem(h.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(), three(1, 1, T), three(0, 0, H), three(0, 0, 1), V, H,
                       -100, H, 0, 0, 0)
    stream = N.raw_stream(0)
    N.check(lib.lvae_vocab_ll_workspace_bytes(q, n))
    ws = N.workspace(n.value, h.device)
    ll, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    N.check(lib.lvae_vocab_ll(q, ll.data_ptr(), lse.data_ptr(), None, None, None, 0, ws.data_ptr(), n.value, stream))
    N.check(lib.lvae_vocab_ll_bwd_workspace_bytes(q, 1, 1, 1, n))
    ws = N.workspace(n.value, h.device)
    got, g = [torch.empty_like(t) for t in (h, w, b)], torch.full((1,), -1.0, device="cuda")
    N.check(lib.lvae_vocab_ll_bwd(q, lse.data_ptr(), g.data_ptr(), three(0, 0, 0), None, None, *[t.data_ptr() for t in got],
                                  ws.data_ptr(), n.value, stream))
    assert torch.equal(ll, D.token_log_likelihood(h, w, y, b))
    for a, e in zip(got, want):
        assert torch.equal(a, e)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_saved_tensors_kept_on_the_host(dt):
    from lvae import decoder_ops as D
    h, w, b, y = (t.cuda() for t in inputs(150, 700, 72, DT[dt]))

    def step():
        ts = [t.clone().requires_grad_() for t in (h, w, b)]
        ll = D.sequence_log_likelihood(ts[0].view(3, 50, 72), ts[1], y.view(3, 50), ts[2])
        return [ll.detach()] + list(torch.autograd.grad(ll.sum(), ts))
    want = step()
    with torch.autograd.graph.save_on_cpu():
        got = step()
    for a, e in zip(got, want):
        assert torch.equal(a, e)


def test_two_captured_steps_that_share_their_memory():
    """Loss, gradients and clipping of a float32 and of a bfloat16 step in two graphs of one pool, replayed in turn."""
    from lvae import decoder_ops as D, grad_ops as G
    data = [tuple(t.cuda() for t in inputs(T, 900, 64, dt, seed=T)) for T, dt in ((200, torch.float32), (40, torch.bfloat16))]

    def step(h, w, b, y):
        ts = [t.detach().requires_grad_() for t in (h, w, b)]
        loss = D.vocab_cross_entropy(ts[0], ts[1], y, ts[2])
        grads = list(torch.autograd.grad(loss, ts))
        norm = G.clip_grads(grads, 0.05)
        return [loss.detach(), norm] + grads
    static = [[t.clone() for t in d] for d in data]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in static:
            step(*s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in static:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=graphs[0].pool() if len(graphs) > 1 else None):
            outs.append(step(*s))
    for k in range(4):
        for i, s in enumerate(static):
            h, _, _, y = (t.cuda() for t in inputs(data[i][0].shape[0], 900, 64, data[i][0].dtype, seed=50 + k, ignore=0.25 * k))
            s[0].copy_(h)
            s[3].copy_(y)
            graphs[i].replay()
            torch.cuda.synchronize()
            want = step(h, data[i][1], data[i][2], y)
            for a, e in zip(outs[i], want):
                assert torch.equal(a, e)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_two_pieces_of_the_vocabulary(dt):
    """More tokens x words than the workspace holds the gradient of at once, the second piece smaller than the first
    (the oracle in float64 on the GPU)."""
    import ctypes
    from lvae import _native as N, decoder_ops as D
    T, V, H = 4096, 70001, 64
    h, w, b, y = (t.cuda() for t in inputs(T, V, H, DT[dt], seed=3))
    gy = torch.randn(T, generator=torch.Generator().manual_seed(1)).cuda()
    three, out = ctypes.c_int64 * 3, ctypes.c_int64(0)
    q = N.VocabProblem(256, 256, 256, 256, three(1, 1, T), three(0, 0, H), three(0, 0, 1), V, H, -100, H, 1 if dt == "bf16" else 0, 0, 0)
    N.check(N.lib().lvae_vocab_ll_bwd_workspace_bytes(q, 0, 1, 0, out))
    assert out.value < T * V * (2 if dt == "bf16" else 4)          # not all of it at once
    ts = [t.clone().requires_grad_() for t in (h, w, b)]
    ll = D.token_log_likelihood(ts[0], ts[1], y, ts[2])
    ll.backward(-gy)
    o = {k: v.cpu() for k, v in oracle(h, w, b, y, gy).items()}
    close(ll, o["ll"], o["tol"], "ll")
    close(ts[0].grad, o["dh"], o["tol_dh"], "d_hidden")
    close(ts[1].grad, o["dw"], o["tol_dw"], "d_weight")
    close(ts[2].grad, o["db"], o["tol_db"], "d_bias")


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_recomputed_in_the_backward(dt, reentrant):
    from torch.utils.checkpoint import checkpoint
    from lvae import decoder_ops as D
    h, w, b, y = (t.cuda() for t in inputs(150, 700, 72, DT[dt]))

    def loss(h, w, b):
        return D.vocab_cross_entropy(h * 2.0, w, y, b)

    def step(f):
        ts = [t.clone().requires_grad_() for t in (h, w, b)]
        out = f(*ts)
        out.backward()
        return [out.detach()] + [t.grad for t in ts]
    for a, e in zip(step(lambda *ts: checkpoint(loss, *ts, use_reentrant=reentrant)), step(loss)):
        assert torch.equal(a, e)


def test_two_host_threads():
    """Calls from two Python threads on streams of their own, errors of one not reported by the other."""
    import threading
    from lvae import decoder_ops as D
    work = [tuple(t.cuda() for t in inputs(T, 2000, 128, dt, seed=T)) for T, dt in ((50, torch.bfloat16), (300, torch.float32))]

    def step(h, w, b, y):
        ts = [t.detach().requires_grad_() for t in (h, w, b)]
        loss = D.vocab_cross_entropy(ts[0], ts[1], y, ts[2])
        return [loss.detach()] + list(torch.autograd.grad(loss, ts))
    want = [step(*x) for x in work]
    torch.cuda.synchronize()
    failures = []

    def run(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = step(*work[k])
                    with pytest.raises(ValueError, match="do not expand"):
                        D.token_log_likelihood(work[k][0], work[k][1], work[k][3][:-1])
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, e) for a, e in zip(got, want[k]))
        except BaseException as e:                        # reported by the main thread
            failures.append(e)
    threads = [threading.Thread(target=run, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
