"""CPU-side checks of the vocabulary and gradient operators: workspace queries, argument checks and refusals, all decided
on the host before anything touches a device."""
import ctypes

import pytest
import torch


def problem(**kw):
    from lvae import _native as N
    three = ctypes.c_int64 * 3
    d = dict(hidden=256, weight=256, bias=None, targets=256, size=three(1, 1, 100), hidden_stride=three(0, 0, 64),
             target_stride=three(0, 0, 1), V=1000, weight_stride=64, ignore_index=-100, H=64, dtype=1, bias_dtype=0, reserved=0)
    d.update(kw)
    return N.VocabProblem(**d)


def test_workspace_queries():
    from lvae import _native as N
    lib, out, three = N.lib(), ctypes.c_int64(0), ctypes.c_int64 * 3
    sizes = []
    for T in (1, 64, 65, 4096):
        assert lib.lvae_vocab_ll_workspace_bytes(problem(size=three(1, 1, T)), out) == 0
        assert out.value > 0 and out.value % 256 == 0
        sizes.append(out.value)
    assert sizes == sorted(sizes)
    assert lib.lvae_vocab_ll_workspace_bytes(problem(), out) == 0
    direct = out.value
    # weights that the tiles cannot read where they lie need a padded copy: odd width, odd pitch, odd address, float32
    for kw in (dict(H=63), dict(weight_stride=65), dict(weight=264), dict(dtype=0)):
        assert lib.lvae_vocab_ll_workspace_bytes(problem(**kw), out) == 0
        assert out.value >= direct + 1000 * 64 * 2, kw
    assert lib.lvae_vocab_ll_bwd_workspace_bytes(problem(), 1, 0, 0, out) == 0
    a = out.value
    assert lib.lvae_vocab_ll_bwd_workspace_bytes(problem(), 1, 1, 1, out) == 0 and out.value >= a
    # the gradient of the logits is bounded, however large tokens x vocabulary gets
    big = problem(size=three(1, 1, 1 << 20), V=200000, H=64)
    assert lib.lvae_vocab_ll_bwd_workspace_bytes(big, 1, 1, 1, out) == 0 and out.value < 8 << 30
    assert lib.lvae_clip_workspace_bytes(0, out) == 0 and out.value > 0
    assert lib.lvae_clip_workspace_bytes(100000, out) == 0 and out.value < 1 << 22


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), b"dtype"), (dict(bias_dtype=-1), b"bias_dtype"), (dict(V=0), b"bad shape"), (dict(H=0), b"bad shape"),
    (dict(H=65537), b"bad shape"), (dict(V=1 << 31), b"bad shape"), (dict(weight_stride=63), b"weight_stride"),
    (dict(size=(ctypes.c_int64 * 3)(1, 0, 5)), b"bad shape"), (dict(size=(ctypes.c_int64 * 3)(65536, 1, 65536)), b"too many")])
def test_problem_refusals(kw, text):
    from lvae import _native as N
    lib, out = N.lib(), ctypes.c_int64(0)
    assert lib.lvae_vocab_ll_workspace_bytes(problem(**kw), out) == -1 and text in lib.lvae_last_error()
    assert lib.lvae_vocab_ll(problem(**kw), 256, None, None, None, None, 0, 256, 1 << 40, None) == -1
    assert lib.lvae_vocab_ll_bwd(problem(**kw), 256, 256, (ctypes.c_int64 * 3)(), None, None, 256, None, None, 256, 1 << 40, None) == -1


@pytest.mark.parametrize("T,V,H,ok", [
    (1, (1 << 26) - 1, 64, True), (1, 1 << 26, 64, False), (1 << 20, 1 << 17, 8191, True), (1 << 20, 1 << 17, 8192, False),
    (1 << 20, (1 << 18) - 1, 64, True), (1 << 20, 1 << 18, 64, False), (1 << 26, 1024, 64, True), (1 << 27, 1024, 8, False)])
def test_limits(T, V, H, ok):
    """Calls whose launches would pass 2^32 threads are refused before the first."""
    from lvae import _native as N
    lib, out, three = N.lib(), ctypes.c_int64(0), ctypes.c_int64 * 3
    q = problem(size=three(1, 1, T), V=V, H=H, weight_stride=H)
    assert (lib.lvae_vocab_ll_workspace_bytes(q, out) == 0) == ok
    assert (lib.lvae_vocab_ll_bwd_workspace_bytes(q, 1, 1, 1, out) == 0) == ok
    assert lib.lvae_vocab_ll_bwd(q, 256, 256, three(), None, None, 256, None, None, 256, 16, None) == (-2 if ok else -1)
    assert lib.lvae_segment_sum_f32(256, 1 << 26, 3, 256, None) == -1


def test_call_refusals():
    from lvae import _native as N
    lib, out, s = N.lib(), ctypes.c_int64(0), (ctypes.c_int64 * 3)()
    assert lib.lvae_vocab_ll_workspace_bytes(None, out) == -1 and lib.lvae_vocab_ll_workspace_bytes(problem(), None) == -1
    for kw in (dict(hidden=None), dict(weight=None), dict(targets=None)):
        assert lib.lvae_vocab_ll(problem(**kw), 256, None, None, None, None, 0, 256, 1 << 40, None) == -1
    assert lib.lvae_vocab_ll(problem(), None, None, None, None, None, 0, 256, 1 << 40, None) == -1
    assert lib.lvae_vocab_ll_workspace_bytes(problem(), out) == 0
    assert lib.lvae_vocab_ll(problem(), 256, None, None, None, None, 0, None, 0, None) == -2 and b"NULL" in lib.lvae_last_error()
    assert lib.lvae_vocab_ll(problem(), 256, None, None, None, None, 0, 260, 1 << 40, None) == -2 and b"aligned" in lib.lvae_last_error()
    assert lib.lvae_vocab_ll(problem(), 256, None, None, None, None, 0, 256, out.value - 1, None) == -2 and b"too small" in lib.lvae_last_error()
    assert lib.lvae_vocab_ll_bwd(problem(), 256, 256, s, None, None, None, None, None, 256, 1 << 40, None) == -1
    assert b"no gradient" in lib.lvae_last_error()
    assert lib.lvae_vocab_ll_bwd(problem(), None, 256, s, None, None, 256, None, None, 256, 1 << 40, None) == -1
    assert lib.lvae_vocab_ll_bwd(problem(), 256, 256, s, None, None, 256, None, None, 256, 16, None) == -2
    assert lib.lvae_vocab_ll(problem(), 256, None, None, 256, None, 1, 256, 1 << 40, None) == -1
    assert b"go together" in lib.lvae_last_error()
    assert lib.lvae_segment_sum_f32(None, 3, 3, 256, None) == -1 and lib.lvae_segment_sum_f32(256, 3, -1, 256, None) == -1


def test_what_a_forward_keeps():
    """float32 tiles keep their exponents and W as two planes of 16 bits, which then need no workspace; nothing else does."""
    from lvae import _native as N
    lib, out, three = N.lib(), ctypes.c_int64(0), ctypes.c_int64 * 3
    for kw, kept in ((dict(dtype=0), 256 + 1000 * 64 * 4), (dict(dtype=0, H=65, weight_stride=70), 256 + 1000 * 128 * 4),
                     (dict(dtype=0, size=three(1, 8, 8)), 0), (dict(dtype=1), 0), (dict(dtype=2, H=63), 0)):
        assert lib.lvae_vocab_ll_kept_bytes(problem(**kw), out) == 0 and out.value == kept, kw
        assert lib.lvae_vocab_ll_workspace_bytes(problem(**kw), out) == 0
        need = out.value - (kept - 256 if kept else 0)
        rc = lib.lvae_vocab_ll(problem(**kw), 256, None, 256, None, None, 0, 256, need - 1, None)
        assert rc == (-2 if kept else -1) and (b"too small" if kept else b"nothing is kept") in lib.lvae_last_error()
        assert lib.lvae_vocab_ll_bwd_workspace_bytes(problem(**kw), 1, 1, 1, out) == 0
        need = out.value - (kept - 256 if kept else 0)
        rc = lib.lvae_vocab_ll_bwd(problem(**kw), 256, 256, three(), None, 256, 256, 256, 256, 256, need - 1, None)
        assert rc == (-2 if kept else -1) and (b"too small" if kept else b"nothing is kept") in lib.lvae_last_error()
    assert lib.lvae_vocab_ll(problem(dtype=0), 256, None, 260, None, None, 0, 256, 1 << 40, None) == -1
    assert b"kept must be 256-byte aligned" in lib.lvae_last_error()
    assert lib.lvae_vocab_ll_kept_bytes(problem(), None) == -1 and lib.lvae_vocab_ll_kept_bytes(problem(V=0), out) == -1


def entries(*rows):
    flat = (ctypes.c_int64 * (4 * len(rows)))()
    for i, (src, dst, n, dt, ot) in enumerate(rows):
        flat[4 * i:4 * i + 4] = [src, dst, n, dt | ot << 32]
    return flat


@pytest.mark.parametrize("rows,text", [
    ([(4096, 0, 10, 0, 0), (4096, 0, 10, 0, 0)], b"share memory"),
    ([(4096, 0, 10, 0, 0), (4100, 0, 10, 0, 0)], b"share memory"),
    ([(8192, 0, 10, 0, 0), (4096, 0, 2000, 0, 0)], b"share memory"),
    ([(4096, 8192, 10, 0, 0), (8200, 16384, 10, 0, 0)], b"share memory"),
    ([(4096, 8192, 10, 0, 0), (16384, 8192, 10, 0, 0)], b"share memory"),
    ([(4096, 4100, 10, 0, 0)], b"share memory"),
    ([(4096, 4096, 10, 0, 1)], b"another type"),
    ([(4096, 0, 10, 3, 0)], b"dtype"), ([(4096, 8192, 10, 0, 7)], b"dtype"),
    ([(0, 0, 10, 0, 0)], b"NULL"), ([(4096, 0, -1, 0, 0)], b"bad size"), ([(4097, 0, 10, 1, 1)], b"aligned")])
def test_list_refusals(rows, text):
    from lvae import _native as N
    lib = N.lib()
    assert lib.lvae_clip_grads(entries(*rows), len(rows), 0, 1, 1.0, 256, 256, 1 << 30, None) == -1
    assert text in lib.lvae_last_error()


def test_clip_call_refusals():
    from lvae import _native as N
    lib, e = N.lib(), entries((4096, 0, 10, 0, 0))
    assert lib.lvae_clip_grads(None, 1, 0, 1, 1.0, 256, 256, 1 << 30, None) == -1
    assert lib.lvae_clip_grads(e, 1, 0, 1, -1.0, 256, 256, 1 << 30, None) == -1
    assert lib.lvae_clip_grads(e, 1, 0, 1, float("nan"), 256, 256, 1 << 30, None) == -1
    assert lib.lvae_clip_grads(e, 1, 0, 1, 1.0, None, 256, 1 << 30, None) == -1
    assert lib.lvae_clip_grads(e, 1, 0, 1, 1.0, 256, None, 1 << 30, None) == -2
    assert lib.lvae_clip_grads(e, 1, 0, 1, 1.0, 256, 260, 1 << 30, None) == -2
    assert lib.lvae_clip_grads(e, 1, 0, 1, 1.0, 256, 256, 16, None) == -2


def test_python_refusals():
    from lvae import _native as N, decoder_ops as D, grad_ops as G
    h, w, y = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    for f in (D.token_log_likelihood, D.vocab_cross_entropy):
        with pytest.raises(N.LvaeError, match="no CPU fallback"):
            f(h, w, y)
        with pytest.raises(N.LvaeError, match="no CPU fallback"):
            f(h.requires_grad_(), w, y)
    with pytest.raises(TypeError):
        D.token_log_likelihood([1.0], w, y)
    with pytest.raises(ValueError, match="sequence axis"):
        D.sequence_log_likelihood(torch.zeros(8), w, y)
    with pytest.raises(ValueError, match="reduction"):
        D.vocab_cross_entropy(h, w, y, reduction="batchmean")
    with pytest.raises(N.LvaeError, match="no CPU fallback"):
        G.global_grad_norm([torch.zeros(3)])
    with pytest.raises(TypeError):
        G.clip_grads([1.0], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        G.clip_grads([], -1.0)


def test_token_axes_are_joined():
    from lvae.decoder_ops import _common_axes
    assert _common_axes((4, 5), [(40, 8), (5, 1)]) == ([1, 1, 20], [[0, 0, 8], [0, 0, 1]])
    assert _common_axes((4, 5), [(48, 8), (5, 1)]) == ([1, 4, 5], [[0, 48, 8], [0, 5, 1]])
    assert _common_axes((2, 3, 4), [(96, 32, 8), (4, 0, 1)]) == ([2, 3, 4], [[96, 32, 8], [4, 0, 1]])
    assert _common_axes((1, 1), [(7, 3), (9, 9)]) == ([1, 1, 1], [[0, 0, 0], [0, 0, 0]])
    assert _common_axes((2, 3, 4, 5), [(1, 2, 6, 24), (60, 20, 5, 1)]) is None
