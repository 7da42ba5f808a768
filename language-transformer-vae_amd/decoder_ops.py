"""The reconstruction half of the objectives: log p(x|z) from a decoder's hidden states.

The reference's decoder multiplies its hidden states with the vocabulary, keeps the ``[batch, seq_len, vocab]`` logits
and calls ``cross_entropy`` on them; the sums over a sentence are the ``log_p_x_z`` of the importance-weighted estimate
(loss_and_optimisation.py:783-794, utils_evaluation.py:176-180).  Here product, softmax and pick are one pass over the
vocabulary (lvae_vocab_ll): no logits exist, forward or backward.

All functions take ``hidden [..., H]`` and ``weight [V, H]`` of one type (float32, bfloat16, float16), an optional
``bias [V]`` of any of these, and ``targets [...]`` (int64) whose shape expands to that of ``hidden`` without its last
axis, so that the ``[B, L]`` words of a batch serve the ``[B, K, L, H]`` states of K latent samples as
``targets[:, None]``.  Positions whose target is ``ignore_index`` count for nothing and cost nothing in the products,
whatever their hidden state holds.  A target outside the vocabulary makes its result, and the gradients it takes part
in, NaN.  A bias of -inf bans a word; hidden states and weights that count have to be finite.  Results are float32, held
and summed in float32 or more; gradients come in the type of what they belong to.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from .estimators import _needs_grad


def _common_axes(shape, strides):
    """The token dimensions as three axes on which every tensor (a list of strides each) steps evenly, or None."""
    axes = []
    for i, n in enumerate(shape):
        if n == 1:
            continue
        here = [s[i] for s in strides]
        if axes and all(p == n * h for p, h in zip(axes[-1][1], here)):
            axes[-1] = (axes[-1][0] * n, here)
        else:
            axes.append((n, here))
    if len(axes) > 3:
        return None
    pad = 3 - len(axes)
    return [1] * pad + [a[0] for a in axes], [[0] * pad + [a[1][k] for a in axes] for k in range(len(strides))]


class _Problem:
    """Checked arguments of one call: the C structure and what keeps its pointers alive."""

    def __init__(self, hidden, weight, targets, bias, ignore_index):
        for t, name in ((hidden, "hidden"), (weight, "weight"), (targets, "targets")) + (((bias, "bias"),) if bias is not None else ()):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
            if not t.is_cuda:
                raise N.LvaeError(f"{name} is on {t.device}: the HIP path needs a GPU tensor (no CPU fallback)")
            if t.device != hidden.device:
                raise ValueError(f"{name} is on {t.device}, hidden on {hidden.device}")
        if hidden.dtype not in N.DTYPES or weight.dtype != hidden.dtype:
            raise TypeError(f"hidden and weight must be of one type, float32, bfloat16 or float16: {hidden.dtype}, {weight.dtype}")
        if bias is not None and bias.dtype not in N.DTYPES:
            raise TypeError(f"bias must be float32, bfloat16 or float16: {bias.dtype}")
        if targets.dtype != torch.int64:
            raise TypeError(f"targets must be int64: {targets.dtype}")
        if hidden.dim() < 1 or weight.dim() != 2 or weight.shape[1] != hidden.shape[-1]:
            raise ValueError(f"shape mismatch: hidden {tuple(hidden.shape)}, weight {tuple(weight.shape)}")
        V, H = weight.shape
        if V < 1 or H < 1:
            raise ValueError(f"weight {tuple(weight.shape)} is empty")
        if bias is not None and bias.shape != (V,):
            raise ValueError(f"bias {tuple(bias.shape)} must be ({V},)")
        self.shape = hidden.shape[:-1]
        if targets.shape != self.shape:
            try:
                targets = targets.expand(self.shape)
            except RuntimeError:
                raise ValueError(f"targets {tuple(targets.shape)} do not expand to {tuple(self.shape)}") from None
        if hidden.stride(-1) != 1 and H > 1:
            hidden = hidden.contiguous()
        if (weight.stride(1) != 1 and H > 1) or (weight.stride(0) < H and V > 1):
            weight = weight.contiguous()
        if bias is not None and not bias.is_contiguous():
            bias = bias.contiguous()
        axes = _common_axes(self.shape, [hidden.stride()[:-1], targets.stride()])
        if axes is None:
            hidden, targets = hidden.contiguous(), targets.contiguous()
            axes = _common_axes(self.shape, [hidden.stride()[:-1], targets.stride()])
        self.tensors = (hidden, weight, targets, bias)
        self.device = hidden.device
        self.T = targets.numel()
        size, (hs, ts) = axes
        three = N._i64 * 3
        self.c = N.VocabProblem(hidden.data_ptr(), weight.data_ptr(), None if bias is None else bias.data_ptr(),
                                targets.data_ptr(), three(*size), three(*hs), three(*ts), V,
                                weight.stride(0) if V > 1 else H, int(ignore_index), H, N.DTYPES[hidden.dtype],
                                0 if bias is None else N.DTYPES[bias.dtype], 0)


def _forward(q, want_lse):
    """(ll, lse or None), both [*token dimensions] float32."""
    dev = q.device
    ll = torch.empty(q.shape, dtype=torch.float32, device=dev)
    lse = torch.empty(q.shape, dtype=torch.float32, device=dev) if want_lse else None
    if q.T:
        nbytes = N._i64(0)
        with torch.cuda.device(dev):
            lib = N.lib()
            N.check(lib.lvae_vocab_ll_workspace_bytes(q.c, nbytes))
            ws = N.workspace(nbytes.value, dev)
            N.check(lib.lvae_vocab_ll(q.c, N.ptr(ll), N.ptr(lse), N.ptr(ws), nbytes.value, N.stream_ptr(dev)))
    return ll, lse


def _backward(q, needs, lse, g, g_axes_strides, g_scale):
    """Gradients of hidden, weight, bias (None where not needed); g is read with the strides given, one per token axis
    of the problem."""
    hidden, weight, _, bias = q.tensors
    dev = q.device
    d_h = torch.empty(hidden.shape, dtype=hidden.dtype, device=dev) if needs[0] else None
    if not q.T:
        return (d_h, torch.zeros(weight.shape, dtype=weight.dtype, device=dev) if needs[1] else None,
                torch.zeros(bias.shape, dtype=bias.dtype, device=dev) if needs[2] else None)
    d_w = torch.empty(weight.shape, dtype=weight.dtype, device=dev) if needs[1] else None
    d_b = torch.empty(bias.shape, dtype=bias.dtype, device=dev) if needs[2] else None
    nbytes = N._i64(0)
    with torch.cuda.device(dev):
        lib = N.lib()
        N.check(lib.lvae_vocab_ll_bwd_workspace_bytes(q.c, int(needs[0]), int(needs[1]), int(needs[2]), nbytes))
        ws = N.workspace(nbytes.value, dev)
        N.check(lib.lvae_vocab_ll_bwd(q.c, N.ptr(lse), N.ptr(g), (N._i64 * 3)(*g_axes_strides), N.ptr(g_scale),
                                      N.ptr(d_h), N.ptr(d_w), N.ptr(d_b), N.ptr(ws), nbytes.value, N.stream_ptr(dev)))
    return d_h, d_w, d_b


def _token_strides(q):
    """Strides of a contiguous [tokens] tensor on the problem's three axes."""
    a, b, c = q.c.size
    return (b * c, c, 1)


# How the log-likelihoods of the tokens are put together: as they are, summed over the last axis, or one loss
_TOKENS, _SEQUENCES, _MEAN, _SUM = range(4)


def _put_together(q, ll, how):
    """(result, device factor of every ll in it or None)."""
    if how == _TOKENS:
        return ll, None
    dev = q.device
    if how == _SEQUENCES:
        out = torch.empty(q.shape[:-1], dtype=torch.float32, device=dev)
        if out.numel():
            with torch.cuda.device(dev):
                N.check(N.lib().lvae_segment_sum_f32(N.ptr(ll), out.numel(), q.shape[-1], N.ptr(out), N.stream_ptr(dev)))
        return out, None
    if not q.T:
        out = torch.zeros(2, dtype=torch.float32, device=dev)
    else:
        out = torch.empty(2, dtype=torch.float32, device=dev)
        with torch.cuda.device(dev):
            N.check(N.lib().lvae_vocab_loss_f32(q.c, N.ptr(ll), int(how == _MEAN), -1.0, N.ptr(out), N.stream_ptr(dev)))
    return out[0], out[1]


class _VocabLL(torch.autograd.Function):
    """Token log-likelihoods, put together, with a HIP backward (lvae_vocab_ll_bwd): the softmax is computed again from
    the saved LSE, a piece of the vocabulary at a time."""

    @staticmethod
    def forward(ctx, hidden, weight, bias, targets, ignore_index, how):
        q = _Problem(hidden.detach(), weight.detach(), targets, None if bias is None else bias.detach(), ignore_index)
        ll, lse = _forward(q, True)
        out, factor = _put_together(q, ll, how)
        ctx.save_for_backward(hidden, weight, bias, targets, lse, factor)
        ctx.ignore_index, ctx.how = ignore_index, how
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        hidden, weight, bias, targets, lse, factor = ctx.saved_tensors
        needs = ctx.needs_input_grad[:3]
        if not any(needs):
            return None, None, None, None, None, None
        q = _Problem(hidden.detach(), weight.detach(), targets, None if bias is None else bias.detach(), ctx.ignore_index)
        if g.dtype != torch.float32:
            g = g.float()
        if ctx.how in (_MEAN, _SUM):
            strides = (0, 0, 0)
        else:
            # sequences: one value for all positions of a sentence; the problem's axes join dimensions, so spread it out
            g = (g if ctx.how == _TOKENS else g.unsqueeze(-1).expand(q.shape)).contiguous()
            strides = _token_strides(q)
        d_h, d_w, d_b = _backward(q, needs, lse, g, strides, factor)
        return d_h, d_w, d_b, None, None, None


def _run(hidden, weight, targets, bias, ignore_index, how):
    if _needs_grad(hidden, weight, bias):
        return _VocabLL.apply(hidden, weight, bias, targets, ignore_index, how)
    det = lambda t: t.detach() if isinstance(t, torch.Tensor) else t
    q = _Problem(det(hidden), det(weight), targets, det(bias), ignore_index)
    return _put_together(q, _forward(q, False)[0], how)[0]


def token_log_likelihood(hidden, weight, targets, bias=None, ignore_index=-100):
    """log p(target | hidden state) of every position, ``[...]`` float32; 0 where the target is ``ignore_index``.
    With up to 64 tokens (a decoding step) the weights are read once, at the speed of memory.  Differentiable in hidden,
    weight and bias."""
    return _run(hidden, weight, targets, bias, ignore_index, _TOKENS)


def sequence_log_likelihood(hidden, weight, targets, bias=None, ignore_index=-100):
    """log p(x|z) of whole sentences: the token log-likelihoods summed over the last axis, ``[...]`` of the axes before
    it.  For hidden ``[B, K, L, H]`` and targets ``[B, 1, L]`` this is the ``log_p_x_z [B, K]`` that ``iw_log_p_x``
    reduces.  A sentence of padding alone has 0.  Differentiable."""
    if isinstance(hidden, torch.Tensor) and hidden.dim() < 2:
        raise ValueError(f"hidden {tuple(hidden.shape)} has no sequence axis")
    return _run(hidden, weight, targets, bias, ignore_index, _SEQUENCES)


def vocab_cross_entropy(hidden, weight, targets, bias=None, ignore_index=-100, reduction="mean"):
    """Cross entropy of the targets, the reconstruction loss of a training step: ``"mean"`` over the positions that
    count (0 if none does), ``"sum"`` over them, or ``"none"`` for every position.  Differentiable."""
    if reduction == "none":
        return -_run(hidden, weight, targets, bias, ignore_index, _TOKENS)
    if reduction not in ("mean", "sum"):
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none': {reduction!r}")
    return _run(hidden, weight, targets, bias, ignore_index, _MEAN if reduction == "mean" else _SUM)
