"""The norm of all gradients together, and clipping by it: what a training step does between backward and update.

Two launches a list of tensors (lvae_clip_grads), and one more for every 112 of a longer one, instead of several for each; the sum of squares is held in float64, and
gradients whose norm is within the bound are not touched.  float32, bfloat16 and float16 gradients may be mixed.
Nothing is copied to or from the host.  Tensors with a forward-mode tangent, torch.func transforms and tracing are refused.
"""
import torch

from . import _native as N

try:
    from . import _tensor_list
except ImportError:                                       # told on the first call, as with liblvae.so
    _tensor_list = None


def _table(src, dst, writes=False):
    if _tensor_list is None:
        raise N.LvaeError("_tensor_list.so is missing: build it with `make -C csrc` (there is no Python fallback)")
    N.check_version("_tensor_list.so", getattr(_tensor_list, "VERSION", None))
    try:
        return _tensor_list.table(src, dst, writes)
    except RuntimeError as e:
        raise N.LvaeError(str(e)) from None


def _call(src, dst, norm_type, scale, max_norm):
    """Norm (and scaling) of the list src, in place or into the list dst; strided tensors go through dense copies."""
    if norm_type not in (2, 2.0, float("inf")):
        raise ValueError(f"norm_type must be 2 or inf: {norm_type!r}")
    table, index, wants_grad, odd = _table(src, dst, scale)
    if index < 0:
        return torch.zeros(())
    if scale and wants_grad and torch.is_grad_enabled():
        raise N.LvaeError("a tensor requires grad: clip gradients, or call under torch.no_grad()")
    copies = dst if dst is not None else src
    if odd:
        src2, copies = list(src), list(copies)
        for i in odd:
            src2[i] = src[i].detach().resolve_neg().contiguous()
            copies[i] = src2[i] if dst is None else torch.empty(dst[i].shape, dtype=dst[i].dtype, device=dst[i].device)
        table = _table(src2, None if dst is None else copies)[0]
    count = len(src)
    nbytes = N._i64(0)
    dev = src[0].device
    with N.on_device(index):
        lib = N.lib()
        N.check(lib.lvae_clip_workspace_bytes(count, nbytes))
        ws = N.workspace(nbytes.value, dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        N.check(lib.lvae_clip_grads(table, count, int(norm_type == float("inf")), int(scale), float(max_norm), norm.data_ptr(),
                                    ws.data_ptr(), nbytes.value, N.raw_stream(index)))
    if scale:
        _tensor_list.written(src if dst is None else dst)
        for i in odd:
            (src if dst is None else dst)[i].detach().copy_(copies[i])
    return norm


def _as_list(tensors):
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def global_grad_norm(grads, norm_type=2.0):
    """Norm over all elements of all tensors, as a 0-dim float32 device tensor: the square root of the sum of squares, or
    with ``norm_type=inf`` the largest magnitude.  NaN where there is one.  Not differentiable."""
    return _call(_as_list(grads), None, norm_type, False, 0.0)


def clip_grads(grads, max_norm, norm_type=2.0, out=None):
    """Scales all gradients by ``min(1, max_norm / (norm + 1e-6))`` and returns their norm before that.  In place; or,
    with ``out`` (one tensor of the same shape for each, of any of the types), into ``out``: 16-bit gradients clipped
    into the float32 buffers of an optimizer are rounded once.  No element that is written may belong to two dense
    tensors, or twice to a broadcast one (LvaeError).  Strided tensors go through dense copies made before anything is
    written, so that the column ranges of one buffer may be listed side by side."""
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative or NaN: {max_norm!r}")
    return _call(_as_list(grads), None if out is None else _as_list(out), norm_type, True, max_norm)


def clip_grad_norm_(parameters, max_norm, norm_type=2.0):
    """``clip_grads`` in place on the ``.grad`` of parameters (those that have one); returns the norm before clipping."""
    parameters = _as_list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    with torch.no_grad():
        return clip_grads(grads, max_norm, norm_type)
