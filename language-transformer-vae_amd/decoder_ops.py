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
derivatives; forward-mode tangents, torch.func transforms and tracing are refused).

What is held in fewer bits: with bfloat16 and float16, the gradient of the logits is rounded to that type once, before the
two products that make the gradients from it.  With float32, more than 64 tokens and any backward multiply operands of 22
bits: an element of hidden, weight or the gradient of the logits below 2^-29 of the largest of its tensor loses bits, and
below 2^-51 of it counts as 0.  The backward of float32 and float16 is held relative to the largest finite upstream
gradient: a position whose own is below 2^-28 of that loses bits of its hidden state's gradient.
"""
import ctypes

import torch

from . import _native as N

try:
    from . import _decoder_calls
except ImportError:                                       # told on the first call, as with liblvae.so
    _decoder_calls = None

_bound = None


def _calls():
    """The C++ side of a call (checks, layout, allocation, launches, autograd), bound to the library that is loaded."""
    global _bound
    lib = N.lib()
    if _bound is not lib:
        if _decoder_calls is None:
            raise N.LvaeError("_decoder_calls.so is missing: build it with `make -C csrc` (there is no Python fallback)")
        N.check_version("_decoder_calls.so", getattr(_decoder_calls, "VERSION", None))
        entry_points = (lib.lvae_vocab_ll_workspace_bytes, lib.lvae_vocab_ll_kept_bytes, lib.lvae_vocab_ll,
                        lib.lvae_vocab_ll_bwd_workspace_bytes, lib.lvae_vocab_ll_bwd, lib.lvae_segment_sum_f32,
                        lib.lvae_last_error)
        _decoder_calls.bind(tuple(ctypes.cast(f, ctypes.c_void_p).value for f in entry_points), N.LvaeError, N.raw_stream)
        _bound = lib
    return _decoder_calls


def _common_axes(shape, strides):
    """The token dimensions as three axes on which every tensor (a list of strides each) steps evenly, or None."""
    return _calls().common_axes(shape, strides)


# How the log-likelihoods of the tokens are put together: as they are, summed over the last axis, or one loss
_TOKENS, _SEQUENCES, _MEAN, _SUM = range(4)


def _run(hidden, weight, targets, bias, ignore_index, how):
    return _calls().log_likelihood(hidden, weight, targets, bias, ignore_index, how)


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
