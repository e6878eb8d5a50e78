"""The global norm of a step's gradients, and the gradients scaled to a largest norm (no counterpart in the
reference, whose trainer clips with torch).

    norm = clip_grads(grads, 1.0)                                  # in place
    norm = clip_grads(grads, 1.0, scale=1.0 / 1024, out=master)    # loss-scaled fp16 into fp32

The norm stays on the device: no call here waits for the GPU.
"""

from array import array
from operator import attrgetter

import torch

from . import _lib

_CODES = {torch.float32: _lib.DK_TYPE_F32, torch.float16: _lib.DK_TYPE_F16,
          torch.bfloat16: _lib.DK_TYPE_BF16}
# a step has hundreds of small gradients: each property is read in the way that takes the least host time
_dtype, _device, _contiguous = attrgetter("dtype"), torch.Tensor.get_device, torch.Tensor.is_contiguous

_OVERLAP = "no gradient may overlap another or be listed twice, and a list holds up to 2^20"


def _dense(t):
    """Whether the tensor's elements fill a run of memory, in whatever order of its axes."""
    expected = 1
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda x: (x[1], x[0])):
        if size != 1:
            if stride != expected:
                return t.numel() == 0
            expected *= size
    return True


def _check(tensors, what):
    """(the tensors' type codes, the device's index)"""
    kinds = set(map(_dtype, tensors))
    if not kinds <= _CODES.keys():
        raise ValueError(f"{what} must be fp32, fp16 or bf16 tensors")
    devices = set(map(_device, tensors))
    if len(devices) != 1 or -1 in devices:
        raise ValueError(f"{what} must be on one GPU")
    if not all(map(_contiguous, tensors)) and not all(map(_dense, tensors)):
        raise ValueError(f"{what} must be dense")
    if len(kinds) == 1:
        codes = array("i", [_CODES[kinds.pop()]]) * len(tensors)
    else:
        codes = array("i", [_CODES[t.dtype] for t in tensors])
    return codes, devices.pop()


def _run(grads, max_norm, scale, out, in_place=False):
    """grads: a list."""
    if not grads:
        raise ValueError("at least one gradient")
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"scale must be positive (got {scale})")
    types, index = _check(grads, "gradients")
    to = types
    # the host arrays live until the call returns
    src, dst = array("q", [g.data_ptr() for g in grads]), None
    numel = array("q", [g.nelement() for g in grads])
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"{len(grads)} gradients, {len(out)} outputs")
        to, there = _check(out, "outputs")
        if there != index or any(
                o.shape != g.shape or (o.stride() != g.stride() and not
                                       (o.is_contiguous() and g.is_contiguous()))
                for o, g in zip(out, grads)):
            raise ValueError("outputs must have their gradients' device, shapes and strides")
        dst = array("q", [o.data_ptr() for o in out])
    elif in_place:
        dst = src
    dev = torch.device("cuda", index)
    lib = _lib.lib()
    nbytes = lib.dk_grad_clip_workspace(len(grads))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    norm = torch.empty_strided((), (), dtype=torch.float32, device=dev)
    try:
        _lib.launch(dev, lib.dk_grad_clip, "dk_grad_clip", src.buffer_info()[0],
                    None if dst is None else dst.buffer_info()[0], numel.buffer_info()[0],
                    types.buffer_info()[0], to.buffer_info()[0], len(grads), max_norm, scale, norm.data_ptr(),
                    ws.data_ptr(), nbytes)
    except ValueError as e:        # (all else that the entry refuses was checked above)
        raise ValueError(f"{_OVERLAP}{'' if out is None else ', outputs included'} ({e})") from None
    return norm


def grad_norm(grads, *, scale=1.0):
    """scale times the 2-norm of all gradients together (fp32 scalar on their device).  grads: CUDA tensors
    (fp32, fp16 or bf16, mixed, dense) of one device; squares are summed in 64 bits."""
    return _run(list(grads), float("inf"), scale, None)


def clip_grads(grads, max_norm, *, scale=1.0, out=None):
    """Scales gradients to a global norm of at most max_norm: with norm = scale * (2-norm of all together)
    each becomes g * scale * min(1, max_norm / (norm + 1e-6)), in place or in `out` (tensors of the
    gradients' shapes, fp32, fp16 or bf16).  Returns the norm before clipping (fp32 scalar on the device).
    An infinite norm scales by 0 and a NaN one gives NaN everywhere (with max_norm infinite only scale counts).
    No tensor may overlap another."""
    if not max_norm > 0.0:
        raise ValueError(f"max_norm must be positive (got {max_norm})")
    return _run(list(grads), max_norm, scale, out, in_place=out is None)


def scale_grads(grads, factor, *, scale=1.0):
    """Each gradient times scale * factor in place; factor: an fp32 scalar tensor on their device, which the
    host does not wait for (the unit of k_loss.row_factors).  No tensor may overlap another, nor hold the
    factor."""
    grads = list(grads)
    if not grads:
        raise ValueError("at least one gradient")
    types, index = _check(grads, "gradients")
    if factor.dtype != torch.float32 or factor.get_device() != index or factor.numel() != 1:
        raise ValueError("factor must be an fp32 scalar on the gradients' device")
    at = array("q", [g.data_ptr() for g in grads])        # (the host arrays live until the call returns)
    numel = array("q", [g.nelement() for g in grads])
    try:
        _lib.launch(torch.device("cuda", index), _lib.lib().dk_grad_scale, "dk_grad_scale", at.buffer_info()[0],
                    numel.buffer_info()[0], types.buffer_info()[0], len(grads), factor.data_ptr(), float(scale))
    except ValueError as e:
        raise ValueError(f"{_OVERLAP}; the factor is in none of them ({e})") from None
