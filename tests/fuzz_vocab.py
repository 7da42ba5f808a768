"""Random shapes through the vocabulary log-likelihoods, forward and backward, against float64 (run by name on a GPU):

    python tests/fuzz_vocab.py [cases] [seed]

How many tokens count is drawn around the places where the tiles change (64, 128, 256 and their multiples), widths and
vocabularies around theirs; types, bias, layouts, upstream gradients and the places of padding at random."""
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "tests")]
from test_gpu_vocab import DT, U, close, oracle  # noqa: E402


def case(rng):
    from lvae import decoder_ops as D
    near = lambda step, top: max(1, step * rng.randint(0, top) + rng.choice((-1, 0, 1, rng.randint(-30, 30))))
    dt = rng.choice(list(DT))
    kept = near(rng.choice((64, 128, 256)), 6)
    T = kept + rng.choice((0, 1, rng.randint(0, 700)))
    V, H = near(rng.choice((64, 256, 1000)), 8), near(rng.choice((8, 64, 128)), 6)
    bias, split = rng.random() < 0.7, rng.choice((1, 1, 2, 3))
    T = -(-T // split) * split
    what = f"dt={dt} kept={kept} T={T} V={V} H={H} bias={bias} split={split}"
    print(what, end=" ", flush=True)
    g = torch.Generator().manual_seed(rng.randrange(1 << 30))
    pitch = H + rng.choice((0, 0, 1, 8))
    h = torch.randn(T, pitch, generator=g)[:, :H].to(DT[dt])
    w = (torch.randn(V, H + rng.choice((0, 0, 3, 8)), generator=g)[:, :H] * 2 / math.sqrt(H)).to(DT[dt])
    b = torch.randn(V, generator=g).to(DT[rng.choice(list(DT))]) if bias else None
    y = torch.randint(0, V, (T,), generator=g)
    y[torch.randperm(T, generator=g)[kept:]] = -100
    gy = torch.randn(T, generator=g) * 10.0 ** rng.randint(-6, 3)
    hc, wc = h.cuda(), w.cuda()
    if rng.random() < 0.3:
        hc[y.cuda() == -100] = math.nan
    o = oracle(h, w, b, y, gy)
    hr, wr, br = hc.requires_grad_(), wc.requires_grad_(), None if b is None else b.cuda().requires_grad_()
    ll = D.token_log_likelihood(hr.view(split, T // split, H) if hr.is_contiguous() else hr, wr,
                                y.cuda().view(split, T // split) if hr.is_contiguous() else y.cuda(), br)
    # The oracle's tolerance grows with the logits alone.  With logits near 0 and many words, |ll| and |LSE| are log V: the
    # logarithm is off by up to a step of it (2 U log V), its sum with the maximum and the subtraction by half a step each
    # (U log V): 4 U log V together, 2.1e-6 for 8,000 words, where the oracle has 2^-20 = 9.5e-7.
    close(ll, o["ll"], o["tol"] + 4 * U * torch.maximum(o["lse"].abs(), o["ll"].abs()), "ll")
    ll.backward(-gy.cuda().view(ll.shape))
    close(hr.grad, o["dh"], o["tol_dh"], "d_hidden")
    close(wr.grad, o["dw"], o["tol_dw"], "d_weight")
    if b is not None:
        close(br.grad, o["db"], o["tol_db"], "d_bias")
    print("ok", flush=True)


def main():
    cases, seed = (int(a) for a in (sys.argv[1:] + ["100", "0"][len(sys.argv) - 1:]))
    rng = random.Random(seed)
    for _ in range(cases):
        case(rng)
    print(f"{cases} cases: clean")


if __name__ == "__main__":
    main()
