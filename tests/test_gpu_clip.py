"""Norm of many gradients and clipping (lvae.grad_ops) against float64.

Tolerances, u = 2^-24: the norm is a float64 sum rounded once, off by u (2u asked); the factor max / (norm + 1e-6) takes
that rounding, its own addition and division (4u), the product one more and the rounding to the result's type half a
step: rel = 6u + eps / 2, plus half of the type's last subnormal step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = [1, 2, 7, 8, 255, 8191, 8192, 8193, 40000]


def tensors(sizes, dts, seed=0, odd=True):
    """Views of one buffer for each type, off the natural alignment."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        dt = DT[dts[i % len(dts)]]
        buf = torch.zeros(n + 3, dtype=dt, device="cuda")
        v = buf[(i % 4 if odd else 0):][:n]
        v.copy_(torch.randn(n, generator=g) * math.exp(i % 3))
        out.append(v)
    return out


def norm64(ts):
    return math.sqrt(sum(t.double().square().sum().item() for t in ts))


def check(got, src, factor, what):
    for i, (a, s) in enumerate(zip(got, src)):
        want = s.double() * factor
        fi = torch.finfo(a.dtype)
        tol = want.abs() * (6 * U + fi.eps / 2) + fi.smallest_normal * fi.eps / 2
        assert ((a.double() - want).abs() <= tol).all(), f"{what}: tensor {i}"


@pytest.mark.parametrize("dts", [["f32"], ["bf16"], ["f16"], ["bf16", "f32", "f16"]])
@pytest.mark.parametrize("copies", [1, 40])
def test_clipped_in_place(dts, copies):
    from lvae import grad_ops as G
    ts = tensors(SIZES * copies, dts)
    src = [t.clone() for t in ts]
    n = norm64(src)
    assert abs(G.global_grad_norm(ts).item() - n) <= 2 * U * n
    norm = G.clip_grads(ts, n / 3)
    assert abs(norm.item() - n) <= 2 * U * n and norm.shape == () and norm.dtype == torch.float32
    check(ts, src, (n / 3) / (n + 1e-6), "in place")


@pytest.mark.parametrize("a,b", [("bf16", "f32"), ("f32", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "f16")])
def test_clipped_into_other_buffers(a, b):
    from lvae import grad_ops as G
    src, out = tensors(SIZES, [a]), tensors(SIZES, [b], seed=4)
    keep = [t.clone() for t in src]
    n = norm64(src)
    G.clip_grads(src, n / 2, out=out)
    check(out, keep, (n / 2) / (n + 1e-6), "out")
    assert all(torch.equal(x, y) for x, y in zip(src, keep))
    G.clip_grads(src, 2 * n, out=out)                # within the bound: copied
    check(out, keep, 1.0, "out, within")


def test_within_the_bound_nothing_changes():
    from lvae import grad_ops as G
    ts = tensors(SIZES, ["f32", "bf16"])
    src = [t.clone() for t in ts]
    n = norm64(src)
    assert abs(G.clip_grads(ts, n * 1.01).item() - n) <= 2 * U * n
    assert all(torch.equal(x, y) for x, y in zip(ts, src))


def test_extremes():
    """Squares beyond float32's range on either side; infinities and NaN; zeros; a bound of zero; nothing at all."""
    from lvae import grad_ops as G
    big = [torch.full((100,), 3e38, device="cuda"), torch.ones(5, device="cuda")]
    assert G.global_grad_norm(big).item() == math.inf          # 3e39 is beyond float32 itself
    big = [torch.full((9,), 1e37, device="cuda")]
    assert abs(G.global_grad_norm(big).item() / 3e37 - 1) < 1e-6
    small = [torch.full((16,), 1e-30, device="cuda")]
    assert abs(G.global_grad_norm(small).item() / 4e-30 - 1) < 1e-6
    z = [torch.zeros(10, device="cuda")]
    assert G.clip_grads(z, 1.0).item() == 0.0 and (z[0] == 0).all()
    t = [torch.ones(10, device="cuda")]
    G.clip_grads(t, 0.0)
    assert (t[0] == 0).all()
    t = [torch.ones(10, device="cuda"), torch.full((9000,), 2.0, device="cuda")]
    t[1][8999] = math.nan
    assert math.isnan(G.clip_grads(t, 1.0).item()) and torch.isnan(t[0]).all()
    t = [torch.ones(10, device="cuda"), torch.full((9000,), 2.0, device="cuda")]
    t[1][17] = -math.inf
    assert G.clip_grads(t, 1.0).item() == math.inf
    assert (t[0] == 0).all() and torch.isnan(t[1][17])          # inf * 0
    assert G.global_grad_norm([]).item() == 0.0
    assert G.global_grad_norm([torch.empty(0, device="cuda")]).item() == 0.0
    e = torch.empty(0, device="cuda")
    assert abs(G.clip_grads([e, torch.ones(4, device="cuda"), e], 5.0).item() - 2.0) < 1e-6


def test_largest_magnitude():
    from lvae import grad_ops as G
    ts = tensors(SIZES, ["f32", "bf16"])
    ts[3][5] = -1234.0          # bfloat16 has steps of 8 between 1024 and 2048: the tensor holds -1232
    assert G.global_grad_norm(ts, norm_type=math.inf).item() == 1232.0
    src = [t.clone() for t in ts]
    G.clip_grads(ts, 617.0, norm_type=math.inf)
    check(ts, src, 617.0 / (1232.0 + 1e-6), "inf norm")
    ts[4][200] = math.nan
    assert math.isnan(G.global_grad_norm(ts, norm_type=math.inf).item())


def test_layouts():
    from lvae import grad_ops as G
    base = torch.randn(40, 50, device="cuda")
    for t in (base.clone().t(), torch.randn(30, 60, device="cuda")[:, ::2], torch.randn(2, 3, 4, 5, device="cuda").permute(0, 2, 3, 1)):
        src = t.clone()
        n = norm64([src])
        assert abs(G.global_grad_norm([t]).item() - n) <= 2 * U * n
        G.clip_grads([t], n / 2)
        check([t], [src], (n / 2) / (n + 1e-6), "strided")
        out = torch.empty(t.shape, device="cuda")
        G.clip_grads([t], n / 4, out=[out])
        check([out], [t], (n / 4) / (norm64([t]) + 1e-6), "strided into dense")


def test_large_tensor_and_captured():
    from lvae import grad_ops as G
    big = torch.randn(30_000_001, device="cuda")[1:]
    ts = [big, torch.randn(77, device="cuda")]
    n = norm64(ts)
    assert abs(G.global_grad_norm(ts).item() - n) <= 2 * U * n
    outs = [torch.empty_like(t) for t in ts]
    G.clip_grads(ts, 1.0, out=outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = G.clip_grads(ts, 1.0, out=outs)
    for k in range(4):
        big.normal_()
        graph.replay()
        torch.cuda.synchronize()
        n = norm64(ts)
        assert abs(norm.item() - n) <= 2 * U * n
        check(outs, ts, 1.0 / (n + 1e-6), "replayed")
        eager = [torch.empty_like(t) for t in ts]
        G.clip_grads(ts, 1.0, out=eager)
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))


def test_refusals():
    from lvae import _native as N, grad_ops as G
    t = torch.ones(100, device="cuda")
    with pytest.raises(N.LvaeError, match="share memory"):
        G.clip_grads([t, t], 1.0)
    with pytest.raises(N.LvaeError, match="share memory"):
        G.clip_grads([t[:60], t[50:]], 1.0)
    with pytest.raises(N.LvaeError, match="share memory"):
        G.clip_grads([t[:50], t[50:]], 1.0, out=[t[50:], torch.empty(50, device="cuda")])
    assert G.global_grad_norm([t, t]).item() == pytest.approx(math.sqrt(200))
    G.clip_grads([t, t], 1.0, out=[torch.empty_like(t), torch.empty_like(t)])      # reading twice is no harm
    assert (t == 1).all()


def test_broadcast_tensors():
    """Read as often as they count; refused, before anything has changed, where they would be written."""
    from lvae import _native as N, grad_ops as G
    a, row = torch.randn(50, device="cuda"), torch.randn(1, 7, device="cuda")
    wide = row.expand(5, 7)
    n = norm64([a, wide])
    assert abs(G.global_grad_norm([a, wide]).item() - n) <= 2 * U * n
    outs = [torch.empty(50, device="cuda"), torch.empty(5, 7, device="cuda")]
    G.clip_grads([a, wide], n / 2, out=outs)
    check(outs, [a, wide], (n / 2) / (n + 1e-6), "broadcast into dense")
    before, version = a.clone(), a._version
    with pytest.raises(N.LvaeError, match=r"grads\[1\] is broadcast"):
        G.clip_grads([a, wide], n / 2)
    with pytest.raises(N.LvaeError, match=r"out\[1\] is broadcast"):
        G.clip_grads([a, wide], n / 2, out=[a, wide])
    assert torch.equal(a, before) and a._version == version


def test_columns_of_one_buffer():
    from lvae import grad_ops as G
    buf = torch.randn(30, 90, device="cuda")
    src, parts = buf.clone(), [buf[:, :40], buf[:, 40:41], buf[:, 41:]]
    n = norm64([src])
    norm = G.clip_grads(parts, n / 3)
    assert abs(norm.item() - n) <= 2 * U * n
    check([buf], [src], (n / 3) / (n + 1e-6), "columns")


@pytest.mark.parametrize("a,b", [("bf16", "f32"), ("f16", None), ("f32", "bf16")])
def test_lists_larger_than_the_caches(a, b):
    """The scaling that goes past the caches, in 16 bits, off the natural alignment and with a ragged end."""
    from lvae import grad_ops as G
    src = [torch.randn(40_000_003, device="cuda").to(DT[a])[3:], torch.randn(1001, device="cuda").to(DT[a])]
    keep = [t.clone() for t in src]
    out = None if b is None else [torch.empty(t.shape, dtype=DT[b], device="cuda") for t in src]
    n = norm64(src)
    norm = G.clip_grads(src, n / 5, out=out)
    assert abs(norm.item() - n) <= 2 * U * n
    check(out or src, keep, (n / 5) / (n + 1e-6), "large")
    if out:
        assert all(torch.equal(x, y) for x, y in zip(src, keep))
