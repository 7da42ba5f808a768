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
and summed in float32 or more; gradients come in the type of what they belong to, and can be taken once (no second
derivatives).  The backward of float32 and float16 is held relative to the largest finite upstream gradient: a position
whose own is below 2^-28 of that loses bits of its hidden state's gradient.
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
        named = [(hidden, "hidden"), (weight, "weight"), (targets, "targets")]
        if bias is not None:
            named.append((bias, "bias"))
        for t, name in named:
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
            if not t.is_cuda:
                raise N.LvaeError(f"{name} is on {t.device}: the HIP path needs a GPU tensor (no CPU fallback)")
        index = hidden.get_device()
        if weight.get_device() != index or targets.get_device() != index or (bias is not None and bias.get_device() != index):
            raise ValueError(f"hidden, weight, targets and bias must be on one device: {[str(t.device) for t, _ in named]}")
        dtype = N.DTYPES.get(hidden.dtype)
        if dtype is None or weight.dtype != hidden.dtype:
            raise TypeError(f"hidden and weight must be of one type, float32, bfloat16 or float16: {hidden.dtype}, {weight.dtype}")
        if bias is not None and bias.dtype not in N.DTYPES:
            raise TypeError(f"bias must be float32, bfloat16 or float16: {bias.dtype}")
        if targets.dtype != torch.int64:
            raise TypeError(f"targets must be int64: {targets.dtype}")
        shape = hidden.shape
        if not shape or weight.dim() != 2 or weight.shape[1] != shape[-1]:
            raise ValueError(f"shape mismatch: hidden {tuple(shape)}, weight {tuple(weight.shape)}")
        V, H = weight.shape
        if V < 1 or H < 1:
            raise ValueError(f"weight {tuple(weight.shape)} is empty")
        if bias is not None and bias.shape != (V,):
            raise ValueError(f"bias {tuple(bias.shape)} must be ({V},)")
        self.shape = shape = shape[:-1]
        if targets.shape != shape:
            try:
                targets = targets.expand(shape)
            except RuntimeError:
                raise ValueError(f"targets {tuple(targets.shape)} do not expand to {tuple(shape)}") from None
        hs, (w0, w1) = hidden.stride(), weight.stride()
        if hs[-1] != 1 and H > 1:
            hidden = hidden.contiguous()
            hs = hidden.stride()
        if (w1 != 1 and H > 1) or (w0 < H and V > 1):
            weight = weight.contiguous()
            w0 = H
        if bias is not None and not bias.is_contiguous():
            bias = bias.contiguous()
        axes = _common_axes(shape, (hs[:-1], targets.stride()))
        if axes is None:
            hidden, targets = hidden.contiguous(), targets.contiguous()
            axes = _common_axes(shape, (hidden.stride()[:-1], targets.stride()))
        self.tensors = (hidden, weight, targets, bias)
        self.layout = _layout(self.tensors)
        self.device, self.index = hidden.device, index
        self.T = targets.numel()
        self.ignore_index = ignore_index
        size, (hs, ts) = axes
        h, w, y, b = _pointers(self.tensors)
        self.c = N.VocabProblem(h, w, b, y, _Three(*size), _Three(*hs), _Three(*ts), V, w0 if V > 1 else H,
                                int(ignore_index), H, dtype, 0 if bias is None else N.DTYPES[bias.dtype], 0)

    def without_tensors(self):
        """(tensors, plan that does not hold them): for the backward, whose tensors autograd keeps."""
        tensors, self.tensors = self.tensors, None
        return tensors, self

    def at(self, tensors):
        """The plan for tensors that autograd has kept: itself, unless a hook of the saved tensors has moved them or laid
        them out anew (even at the old address: the memory may have been free in between)."""
        if _layout(tensors) == self.layout:
            return self
        h, w, y, b = tensors
        return _Problem(h, w, y, b, self.ignore_index)


_Three = N._i64 * 3


def _pointers(tensors):
    return [None if t is None else t.data_ptr() for t in tensors]


def _layout(tensors):
    return [None if t is None else (t.data_ptr(), t.stride()) for t in tensors]


# How the log-likelihoods of the tokens are put together: as they are, summed over the last axis, or one loss
_TOKENS, _SEQUENCES, _MEAN, _SUM = range(4)


def _forward(q, how, for_backward):
    """(result, what the backward needs): the latter the LSE of every token, the factor of every token in a loss, and the
    exponents of float32 operands; each None where there is none."""
    dev = q.device
    ll = torch.empty(q.shape, dtype=torch.float32, device=dev)
    lse = torch.empty(q.shape, dtype=torch.float32, device=dev) if for_backward else None
    limbs = for_backward and q.T > N.VOCAB_FEW and q.c.dtype == N.DTYPES[torch.float32]
    exponents = torch.empty(2, dtype=torch.int32, device=dev) if limbs else None
    loss = each = None
    if how >= _MEAN:
        new = torch.empty if q.T else torch.zeros
        loss, each = new((), dtype=torch.float32, device=dev), new((), dtype=torch.float32, device=dev)
    out = ll if loss is None else loss
    if how == _SEQUENCES:
        out = torch.empty(q.shape[:-1], dtype=torch.float32, device=dev)
    if q.T or (how == _SEQUENCES and out.numel()):
        lib = N.lib()
        with N.on_device(q.index):
            stream = N.raw_stream(q.index)
            if q.T:
                nbytes = N._i64(0)
                N.check(lib.lvae_vocab_ll_workspace_bytes(q.c, nbytes))
                ws = N.workspace(nbytes.value, dev)
                N.check(lib.lvae_vocab_ll(q.c, *_pointers((ll, lse, exponents, loss, each)), how == _MEAN, ws.data_ptr(),
                                          nbytes.value, stream))
            if how == _SEQUENCES and out.numel():
                N.check(lib.lvae_segment_sum_f32(ll.data_ptr(), out.numel(), q.shape[-1], out.data_ptr(), stream))
    return out, (lse, each, exponents)


def _backward(q, tensors, needs, lse, g, g_strides, g_scale, exponents):
    """Gradients of hidden, weight, bias (None where not needed); g is read with the strides given, one per token axis
    of the problem."""
    hidden, weight, _, bias = tensors
    dev = q.device
    new = torch.empty if q.T else torch.zeros
    d_h = torch.empty(hidden.shape, dtype=hidden.dtype, device=dev) if needs[0] else None
    d_w = new(weight.shape, dtype=weight.dtype, device=dev) if needs[1] else None
    d_b = new(bias.shape, dtype=bias.dtype, device=dev) if needs[2] else None
    if q.T:
        nbytes = N._i64(0)
        with N.on_device(q.index):
            lib = N.lib()
            N.check(lib.lvae_vocab_ll_bwd_workspace_bytes(q.c, needs[0], needs[1], needs[2], nbytes))
            ws = N.workspace(nbytes.value, dev)
            p = _pointers((lse, g, g_scale, exponents, d_h, d_w, d_b))
            N.check(lib.lvae_vocab_ll_bwd(q.c, p[0], p[1], _Three(*g_strides), *p[2:], ws.data_ptr(), nbytes.value,
                                          N.raw_stream(q.index)))
    return d_h, d_w, d_b


def _token_strides(q):
    """Strides of a contiguous [tokens] tensor on the problem's three axes."""
    _, b, c = q.c.size
    return (b * c, c, 1)


class _VocabLL(torch.autograd.Function):
    """Token log-likelihoods, put together, with a HIP backward (lvae_vocab_ll_bwd): the softmax is computed again from
    the saved LSE, a piece of the vocabulary at a time."""

    @staticmethod
    def forward(ctx, hidden, weight, bias, targets, ignore_index, how):
        q = _Problem(hidden.detach(), weight.detach(), targets, None if bias is None else bias.detach(), ignore_index)
        out, saved = _forward(q, how, True)
        tensors, ctx.plan = q.without_tensors()
        ctx.save_for_backward(*tensors, *saved)
        ctx.how = how
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        *tensors, lse, factor, exponents = ctx.saved_tensors
        needs = ctx.needs_input_grad[:3]
        if not any(needs):
            return None, None, None, None, None, None
        q = ctx.plan.at(tensors)
        if g.dtype != torch.float32:
            g = g.float()
        if ctx.how >= _MEAN:
            strides = (0, 0, 0)
        else:
            # sequences: one value for all positions of a sentence; the problem's axes join dimensions, so spread it out
            g = (g if ctx.how == _TOKENS else g.unsqueeze(-1).expand(q.shape)).contiguous()
            strides = _token_strides(q)
        return (*_backward(q, tensors, needs, lse, g, strides, factor, exponents), None, None, None)


def _run(hidden, weight, targets, bias, ignore_index, how):
    if _needs_grad(hidden, weight, bias):
        return _VocabLL.apply(hidden, weight, bias, targets, ignore_index, how)
    q = _Problem(hidden, weight, targets, bias, ignore_index)
    return _forward(q, how, False)[0]


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
