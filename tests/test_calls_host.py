"""CPU-side checks of what the vocabulary and gradient operators refuse before they ask where a tensor lives."""
import pytest
import torch
import torch.autograd.forward_ad as fwd


def arguments():
    return torch.randn(3, 8), torch.randn(5, 8), torch.randn(5), torch.zeros(3, dtype=torch.int64)


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(which, grad):
    """The kernels read memory and carry no tangent: a result without one would count as a derivative of zero."""
    from lvae import _native as N, decoder_ops as D, grad_ops as G
    h, w, b, y = arguments()
    ts = [h, w, b]
    if grad:
        ts[which].requires_grad_()
    with fwd.dual_level():
        dual = list(ts)
        dual[which] = fwd.make_dual(ts[which], torch.ones_like(ts[which]))
        for f in (D.token_log_likelihood, D.sequence_log_likelihood, D.vocab_cross_entropy):
            with pytest.raises(N.LvaeError, match="forward-mode"):
                f(dual[0], dual[1], y, dual[2])
            with torch.no_grad(), pytest.raises(N.LvaeError, match="forward-mode"):
                f(dual[0], dual[1], y, dual[2])
        for f in (G.global_grad_norm, lambda t: G.clip_grads(t, 1.0)):
            with pytest.raises(N.LvaeError, match="forward-mode"):
                f([dual[which]])
    with pytest.raises(N.LvaeError, match="no CPU fallback"):     # the tangent has gone with its level
        D.token_log_likelihood(dual[0], dual[1], y, dual[2])


def test_transforms_are_refused():
    """torch.func wraps its tensors: they have no memory of their own."""
    from lvae import _native as N, decoder_ops as D, grad_ops as G
    h, w, b, y = arguments()
    loss = lambda h: D.vocab_cross_entropy(h, w, y, b)
    with pytest.raises(N.LvaeError, match="torch.func"):
        torch.func.grad(loss)(h)
    with pytest.raises(N.LvaeError, match="torch.func"):
        torch.func.jvp(loss, (h,), (h,))
    with pytest.raises(N.LvaeError, match="torch.func"):
        torch.func.vmap(loss)(h[None])
    with pytest.raises(N.LvaeError, match="torch.func"):
        torch.func.vmap(lambda y: D.token_log_likelihood(h, w, y, b))(y[None])
    with pytest.raises(N.LvaeError, match="torch.func"):
        torch.func.vmap(lambda t: G.global_grad_norm([t]))(h)


@pytest.mark.parametrize("grad", [False, True])
def test_tracing_is_refused(grad):
    """A trace would hold the allocations and not the kernels."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch._subclasses.fake_tensor import FakeTensorMode
    from lvae import _native as N, decoder_ops as D, grad_ops as G
    h, w, b, y = arguments()
    h.requires_grad_(grad)
    calls = [(lambda h: D.token_log_likelihood(h, w, y, b), h), (lambda h: D.vocab_cross_entropy(h, w, y, b), h),
             (lambda t: G.global_grad_norm([t]), w), (lambda t: G.clip_grads([t], 1.0), w)]
    for f, x in calls:
        with pytest.raises(N.LvaeError, match="traced"):
            torch.jit.trace(f, (x,))
        with pytest.raises(N.LvaeError, match="traced"):
            make_fx(f)(x)
        with FakeTensorMode() as fake, pytest.raises(N.LvaeError, match="traced"):
            f(fake.from_tensor(x))


@pytest.mark.parametrize("source", ["grad_clip", "vocab_ce", "vocab_tiles_f32", "vocab_tiles_bf16", "vocab_tiles_f16"])
def test_no_kernel_promises_an_alignment_that_its_callers_need_not_have(source):
    """Tensors are views that start anywhere: an access through a pointer that has lost its reduced alignment on the way
    promises the compiler 8 or 16 bytes.  The compiler's own diagnosis, as an error."""
    import os
    import subprocess
    hipcc = "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no HIP compiler")
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "language-transformer-vae_amd", "csrc")
    r = subprocess.run([hipcc, "-std=c++17", "--offload-arch=gfx950", "-fsyntax-only", "-Werror=align-mismatch", source + ".hip"],
                       cwd=csrc, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]


def test_the_libraries_say_what_they_were_built_from():
    from lvae import _decoder_calls, _native as N, _tensor_list
    import os
    import re
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "lvae.h")).read()
    assert int(re.search(r"#define LVAE_VERSION (\d+)", header).group(1)) == N.VERSION == N.lib().lvae_version()
    assert _decoder_calls.VERSION == _tensor_list.VERSION == N.VERSION


def test_a_library_of_another_version_is_refused(tmp_path, monkeypatch):
    """Before anything is called with arguments that it would take for others."""
    import os
    import subprocess
    import sys
    import types
    from lvae import _native as N, decoder_ops as D, grad_ops as G
    (tmp_path / "old.c").write_text("int lvae_version(void) { return 100; }\n")
    subprocess.run(["gcc", "-shared", "-fPIC", "old.c", "-o", "old.so"], cwd=tmp_path, check=True)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", "from lvae import _native as N\ntry: N.lib()\nexcept N.LvaeError as e: print('refused:', e)"],
                       cwd=root, env=dict(os.environ, LVAE_LIB=str(tmp_path / "old.so")), capture_output=True, text=True, timeout=300)
    assert r.stdout.startswith("refused:") and "is of version 100" in r.stdout, r.stdout + r.stderr
    old = types.SimpleNamespace(bind=None, log_likelihood=None, table=None)       # an extension from before it said so
    monkeypatch.setattr(D, "_decoder_calls", old)
    monkeypatch.setattr(D, "_bound", None)
    monkeypatch.setattr(G, "_tensor_list", old)
    h, w, b, y = arguments()
    with pytest.raises(N.LvaeError, match="_decoder_calls.so is of version None"):
        D.token_log_likelihood(h, w, y, b)
    with pytest.raises(N.LvaeError, match="_tensor_list.so is of version None"):
        G.global_grad_norm([h])


def test_the_c_library_builds_without_python_and_torch():
    """`make` (dry run) of a user of the C ABI alone."""
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "language-transformer-vae_amd", "csrc")

    def commands(*args):
        r = subprocess.run(["make", "-n", "-B", "-C", csrc, *args], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stderr
        assert "-o ../liblvae.so" in r.stdout
        return r
    for args in (["PYTHON=/nonexistent/python3"], ["lib"], ["lib", "PYTHON=/nonexistent/python3"]):
        r = commands(*args)
        assert "_decoder_calls.cpp" not in r.stdout and "python3.1" not in r.stdout
        assert "decoder_calls.cpp -o" not in r.stdout and "No such file" not in r.stderr
    assert "decoder_calls.cpp -o" in commands().stdout and "tensor_list.cpp -o" in commands().stdout
