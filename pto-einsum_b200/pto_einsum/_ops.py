"""Calls into the core library for operators that take strided torch tensors: argument
structs, streams and the checks they share."""
from __future__ import annotations

import ctypes
import struct

import torch
from torch.autograd import forward_ad

from ._core import core_lib, error_string
from .builder import _raw_stream_getter

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

_get_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_raw_stream = None
_fns: dict = {}


# Argument checks and layouts of earlier calls, by signature: the shapes, strides, types
# and devices of the tensors (never their addresses or values). A call whose signature
# is here needs no further checks; only calls that copy nothing are kept.
_MOST_PLANS = 4096
_plans: dict = {}


def sig(t):
    """What a plan may depend on of a tensor."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def sigs(*tensors):
    """That of several, and where gradients are recorded whether they ask for one."""
    if not torch.is_grad_enabled():
        return tuple([None if t is None else (t.shape, t.stride(), t.dtype, t.get_device()) for t in tensors])
    return tuple([None if t is None else (t.shape, t.stride(), t.dtype, t.get_device(), t.requires_grad)
                  for t in tensors])


def plan(key):
    return _plans.get(key)


def keep_plan(key, value):
    if len(_plans) >= _MOST_PLANS:
        _plans.clear()
    _plans[key] = value
    return value


def packer(fields: str) -> struct.Struct:
    """An argument struct of 8-byte fields: q integers, Q pointers, d doubles."""
    return struct.Struct("=" + fields)


def function(name: str, restype=ctypes.c_int, argtypes=(ctypes.c_char_p, ctypes.c_void_p)):
    """The core library's `name`; the operators take (argument struct, stream)."""
    fn = _fns.get(name)
    if fn is None:
        fn = getattr(core_lib(), name)
        fn.argtypes, fn.restype = list(argtypes), restype
        _fns[name] = fn
    return fn


def call(name: str, args: bytes, idx: int):
    """Enqueue on the current stream of device `idx`; a nonzero status raises RuntimeError."""
    global _raw_stream
    fn = _fns.get(name) or function(name)
    if idx == _get_device():
        if _raw_stream is None:
            _raw_stream = _raw_stream_getter()
        rc = fn(args, _raw_stream(idx))
    else:
        with torch.cuda.device(idx):
            rc = fn(args, torch.cuda.current_stream(idx).cuda_stream)
    if rc:
        raise RuntimeError(f"pto_einsum: {name} failed: {error_string(rc)} ({rc})")


def sized(name: str, args: bytes, idx: int) -> int:
    """Workspace bytes; the rule may ask the device for its number of SMs."""
    fn = _fns.get(name) or function(name, ctypes.c_int64, (ctypes.c_char_p,))
    if idx == _get_device():
        return fn(args)
    with torch.cuda.device(idx):
        return fn(args)


_sizes: dict = {}


def nbytes_of(name: str, lay, args) -> int:
    """Workspace bytes of a call with this layout: they depend on its numbers alone."""
    key = (name, lay[0], lay[2])
    n = _sizes.get(key)
    if n is None:
        if len(_sizes) >= _MOST_PLANS:
            _sizes.clear()
        n = _sizes[key] = sized(name, args(), lay[2])
    return n


def empty(t):
    """A contiguous tensor of t's shape, type and device."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def workspace(nbytes: int, dev: torch.device):
    """Scratch from torch's caching allocator, so it belongs to the current stream."""
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def check_tensor(name: str, t, shape, dtype, dev):
    """`t` must be a tensor of that shape, type and device."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor (got {type(t).__name__})")
    if t.device != dev:
        raise ValueError(f"{name} must be on {dev} (got {t.device})")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype} (got {t.dtype})")
    if t.shape != torch.Size(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)} (got {tuple(t.shape)})")


def check_activations(name: str, t, dims):
    """The tensor whose type and device the others follow."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor (got {type(t).__name__})")
    if t.device.type != "cuda":
        raise ValueError(f"pto_einsum: {name} must be a CUDA tensor (got {t.device})")
    if t.dtype not in DTYPES:
        raise TypeError(f"{name} must be float32, float16 or bfloat16 (got {t.dtype})")
    if t.dim() not in dims:
        raise ValueError(f"{name} must have {' or '.join(map(str, dims))} dimensions (got shape {tuple(t.shape)})")


def rows(t):
    """`t` with a last axis of stride 1 (a copy where it has another)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def stride(t, axis: int) -> int:
    """Stride of an axis, 0 for one of length one (whatever the tensor says of it)."""
    return 0 if t is None or t.shape[axis] == 1 else t.stride(axis)


def offsets(cu_seqlens, batch: int, tokens: int, dev):
    """cu_seqlens as an int32 tensor on `dev`, and the number of sequences.

    A list or a host tensor is checked here; one on the device is not read by the host
    (the kernels keep within the tensors whatever it holds and report a wrong table in
    the device error word)."""
    if cu_seqlens is None:
        return None, batch
    if batch != 1:
        raise ValueError(f"cu_seqlens takes one row of packed sequences (got a batch of {batch})")
    if tokens > 2 ** 31 - 1:
        raise ValueError("cu_seqlens takes rows of less than 2**31 tokens")
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.device.type == "cpu":
        given = list(cu_seqlens.tolist() if hasattr(cu_seqlens, "tolist") else cu_seqlens)
        cu = [int(v) for v in given]
        if cu != given:
            raise ValueError("cu_seqlens must be whole numbers")
        if len(cu) < 2 or cu[0] != 0 or cu[-1] != tokens or any(a > b for a, b in zip(cu, cu[1:])):
            raise ValueError(f"cu_seqlens must rise from 0 to the {tokens} tokens of the row")
        return torch.tensor(cu, dtype=torch.int32, device=dev), len(cu) - 1
    if cu_seqlens.device != dev:
        raise ValueError(f"cu_seqlens must be on {dev} (got {cu_seqlens.device})")
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2:
        raise ValueError(f"cu_seqlens must be one row of at least two offsets (got {tuple(cu_seqlens.shape)})")
    if cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"cu_seqlens must be int32 or int64 (got {cu_seqlens.dtype})")
    if cu_seqlens.dtype == torch.int64:      # an offset past the row stays past it, and is reported
        cu_seqlens = cu_seqlens.clamp(-1, min(tokens + 1, 2 ** 31 - 1))
    return cu_seqlens.to(torch.int32).contiguous(), cu_seqlens.shape[0] - 1   # itself if it is that


def check_slots(slots, batch: int, dev):
    if slots is None:
        return
    if not isinstance(slots, torch.Tensor) or slots.dtype not in (torch.int32, torch.int64):
        raise TypeError("slots must be an int32 or int64 tensor")
    if slots.device != dev or slots.shape != (batch,) or (batch > 1 and slots.stride(0) != 1):
        raise ValueError(f"slots must be a contiguous tensor of {batch} indices on {dev}")


def slot_pointers(slots):
    """(pointer to int32 slots, pointer to int64 slots)."""
    if slots is None:
        return 0, 0
    return (slots.data_ptr(), 0) if slots.dtype == torch.int32 else (0, slots.data_ptr())


def wants_grad(*tensors) -> bool:
    """Whether autograd has to see the call: gradients are recorded for an input, or one
    carries a tangent (forward mode, which no_grad leaves on)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if forward_ad._current_level >= 0:   # inside dual_level
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                return True
    return False
