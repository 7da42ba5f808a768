"""The norm of all gradients together, and clipping by it: what a training step does between backward and update.

Two launches a list of tensors (lvae_clip_grads) instead of several for each; the sum of squares is held in float64, and
gradients whose norm is within the bound are not touched.  float32, bfloat16 and float16 gradients may be mixed.
Nothing is copied to or from the host.
"""
import array

import torch

from . import _native as N


def _dense(t):
    """Whether the elements of t fill one stretch of memory, each once, in whatever order of the axes."""
    step = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if s != step:
            return False
        step *= n
    return True


def _list(tensors, name):
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    for i, t in enumerate(tensors):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}[{i}] must be a torch.Tensor")
        if not t.is_cuda:
            raise N.LvaeError(f"{name}[{i}] is on {t.device}: the HIP path needs a GPU tensor (no CPU fallback)")
        if t.dtype not in N.DTYPES:
            raise TypeError(f"{name}[{i}] must be float32, bfloat16 or float16: {t.dtype}")
        if t.device != tensors[0].device:
            raise ValueError(f"{name}[{i}] is on {t.device}, {name}[0] on {tensors[0].device}: one device a call")
    return tensors


def _call(src, dst, norm_type, scale, max_norm):
    """src: dense tensors; dst: matching tensors or None for in place."""
    if norm_type not in (2, 2.0, float("inf")):
        raise ValueError(f"norm_type must be 2 or inf: {norm_type!r}")
    if not src:
        return torch.zeros(())
    dev = src[0].device
    flat = array.array("q")
    codes = N.DTYPES
    for t, d in zip(src, dst or src):
        flat.extend((t.data_ptr(), d.data_ptr() if dst else 0, t.numel(), codes[t.dtype] | codes[d.dtype] << 32))
    count = len(src)
    nbytes = N._i64(0)
    with torch.cuda.device(dev):
        lib = N.lib()
        N.check(lib.lvae_clip_workspace_bytes(count, nbytes))
        ws = N.workspace(nbytes.value, dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        N.check(lib.lvae_clip_grads(flat.buffer_info()[0], count, int(norm_type == float("inf")), int(scale), float(max_norm),
                                    N.ptr(norm), N.ptr(ws), nbytes.value, N.stream_ptr(dev)))
    return norm


def global_grad_norm(grads, norm_type=2.0):
    """Norm over all elements of all tensors, as a 0-dim float32 device tensor: the square root of the sum of squares, or
    with ``norm_type=inf`` the largest magnitude.  NaN where there is one."""
    src = [t.detach() if t.is_contiguous() or _dense(t) else t.detach().contiguous() for t in _list(grads, "grads")]
    return _call(src, None, norm_type, False, 0.0)


def clip_grads(grads, max_norm, norm_type=2.0, out=None):
    """Scales all gradients by ``min(1, max_norm / (norm + 1e-6))`` and returns their norm before that.  In place; or,
    with ``out`` (one tensor of the same shape for each, of any of the types), into ``out``: 16-bit gradients clipped
    into the float32 buffers of an optimizer are rounded once.  No element that is written may belong to two of the
    tensors (LvaeError)."""
    src = _list(grads, "grads")
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative or NaN: {max_norm!r}")
    if any(t.requires_grad for t in src) and torch.is_grad_enabled():
        raise N.LvaeError("a tensor requires grad: clip gradients, or call under torch.no_grad()")
    if out is None:
        odd = [i for i, t in enumerate(src) if not t.is_contiguous() and not _dense(t)]
        if not odd:
            return _call(src, None, norm_type, True, max_norm)
        dense = list(src)
        for i in odd:                       # strided gradients go through a dense copy
            dense[i] = src[i].contiguous()
        norm = _call(dense, None, norm_type, True, max_norm)
        for i in odd:
            src[i].copy_(dense[i])
        return norm
    dst = _list(out, "out")
    if len(dst) != len(src):
        raise ValueError(f"{len(src)} gradients, {len(dst)} tensors in out")
    for i, (t, d) in enumerate(zip(src, dst)):
        if t.shape != d.shape:
            raise ValueError(f"out[{i}] is {tuple(d.shape)}, grads[{i}] {tuple(t.shape)}")
        if d.device != t.device:
            raise ValueError(f"out[{i}] is on {d.device}, grads[{i}] on {t.device}")
    # the same order of elements on both sides; any other layout through dense copies
    plain = lambda t, d: t.stride() == d.stride() and (t.is_contiguous() or _dense(t)) or (t.is_contiguous() and d.is_contiguous())
    odd = [i for i, (t, d) in enumerate(zip(src, dst)) if not plain(t, d)]
    s2, d2 = list(src), list(dst)
    for i in odd:
        s2[i], d2[i] = src[i].contiguous(), torch.empty(dst[i].shape, dtype=dst[i].dtype, device=dst[i].device)
    norm = _call(s2, d2, norm_type, True, max_norm)
    for i in odd:
        dst[i].copy_(d2[i])
    return norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0):
    """``clip_grads`` in place on the ``.grad`` of parameters (those that have one); returns the norm before clipping."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = [p.grad for p in parameters if p.grad is not None]
    with torch.no_grad():
        return clip_grads(grads, max_norm, norm_type)
