"""Loads libvgpu_ops.so (csrc/ops/*.hip) and holds its argument structures.

The library is built in-tree by ``make native``.  On a GPU there is no other
path: a missing library is an error, never a silent fallback.
"""
from __future__ import annotations

import ctypes
from ctypes import POINTER, c_float, c_int32, c_int64, c_uint64, c_void_p
from functools import lru_cache
from pathlib import Path

import torch
from torch.autograd import forward_ad
from torch.utils._device import DeviceContext

PACKAGE = Path(__file__).resolve().parent.parent
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_PLAIN_TENSORS = (torch.Tensor, torch.nn.Parameter)


def _struct(name, **groups):
    fields = [(f, kind) for kind, names in groups.values() for f in names.split()]
    return type(name, (ctypes.Structure,), {"_fields_": fields})


LinearArgs = _struct(
    "LinearArgs", a=(c_void_p, "x w bias res dy y z dx dw db work"),
    b=(c_int64, "m n k xs0 xs1 ws0 ws1 ldr lddy work_bytes"), c=(c_int32, "dtype act"))
NormArgs = _struct(
    "NormArgs", a=(c_void_p, "x weight bias dy y dx dweight dbias mean rstd part"),
    b=(c_int64, "ldx ldy lddy lddx rows groups d"), c=(c_int32, "dtype wtype parts"),
    d=(c_float, "eps"))
DistillArgs = _struct(
    "DistillArgs",
    a=(c_void_p, "x index teacher dx grad rows_loss state origin most log_sum slot_p loss counts slot_i "
                 "part"),
    b=(c_int64, "ldx lddx ldi ldt rows v"),
    c=(c_int32, "dtype ttype index_bytes top chunks reduction written"), d=(c_float, "temperature scale"))


@lru_cache(maxsize=None)
def library() -> ctypes.CDLL:
    # torch has loaded its HIP runtime by now; the library binds to that one
    # by its soname, so streams and memory are shared
    for path in (PACKAGE / "csrc" / "libvgpu_ops.so", PACKAGE.parent / "lib" / "libvgpu_ops.so"):
        if path.exists():
            break
    else:
        raise RuntimeError(
            "libvgpu_ops.so is not built: run `make native` (hipcc, gfx950)")
    lib = ctypes.CDLL(str(path))
    for name, struct in (("linear", LinearArgs), ("norm", NormArgs), ("distill", DistillArgs)):
        getattr(lib, "vgpu_ops_" + name).argtypes = [POINTER(struct), c_void_p]
    lib.vgpu_ops_linear_work.argtypes = [POINTER(LinearArgs)]
    lib.vgpu_ops_linear_work.restype = c_int64
    lib.vgpu_ops_norm_parts.argtypes = [c_int64, c_int64, c_int64]
    lib.vgpu_ops_capture.argtypes = [c_void_p]
    lib.vgpu_ops_capture.restype = c_uint64
    lib.vgpu_ops_distill_chunks.argtypes = [c_int64, c_int64, c_int32]
    return lib


def on_gpu(*tensors) -> bool:
    """Whether the kernels run: ordinary tensors on a GPU, and nothing that
    traces or transforms the call.  Otherwise the plain formula runs: so too
    for tensors whose sign is still to be turned, as conj()'s imaginary part,
    inside forward-mode differentiation, and under a mode that records, counts
    or replaces torch's operations and would miss the call."""
    if (torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack()
            or (torch._C._len_torch_function_stack() and _watched())):
        return False
    for t in tensors:
        if t is not None and (type(t) not in _PLAIN_TENSORS or not t.is_cuda or t.is_neg()):
            return False
    return not (torch._C._get_tracing_state() is not None
                or torch._C._are_functorch_transforms_active()
                or forward_ad._current_level >= 0)


def _watched() -> bool:
    """Whether a function mode looks on, other than the default device's."""
    return any(type(mode) is not DeviceContext
               for mode in torch.overrides._get_current_function_mode_stack())


_entries = {}   # name -> bound function
_devices = set()  # whose architecture has been looked at


def entry(name: str):
    found = _entries.get(name)
    if found is None:
        found = _entries[name] = getattr(library(), "vgpu_ops_" + name)
    return found


def _look_at(index):
    arch = torch.cuda.get_device_properties(index).gcnArchName
    if not arch.startswith("gfx950"):
        raise RuntimeError(f"the head operators are built for gfx950, not {arch}")
    _devices.add(index)


def launch(name: str, device: torch.device, *args) -> None:
    """Runs an entry point on the device's current stream."""
    index = device.index
    if index not in _devices:
        _look_at(index)
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return launch(name, device, *args)
    rc = entry(name)(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        raise RuntimeError(f"vgpu_ops_{name}: " + ("refused the arguments" if rc < 0
                                                   else f"HIP error {rc}"))


def capture(device: torch.device) -> int:
    """The number of the capture that the device's current stream takes part
    in, 0 for none (as of the default stream, which cannot)."""
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    return entry("capture")(stream) if stream else 0


@lru_cache(maxsize=4096)
def plan(name: str, *sizes) -> int:
    """What a launch of these sizes needs; a function of the sizes alone."""
    return entry(name)(*sizes)


def autocast(device: torch.device) -> bool:
    return (torch._C._is_any_autocast_enabled() and device.type in ("cuda", "cpu")
            and torch.is_autocast_enabled(device.type))


def needs_grad(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def rows_of(t: torch.Tensor, width: int) -> torch.Tensor:
    """[..., width] as a matrix whose rows are contiguous."""
    m = t if t.dim() == 2 else t.reshape(-1, width)
    return m if width == 1 or m.stride(1) == 1 else m.contiguous()


def ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def same_device(names: str, first, *others) -> None:
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            raise ValueError("tensors on different devices: " + ", ".join(
                f"{n} on {t.device}" for n, t in zip(names.split(), (first, *others))
                if t is not None))


def formula_backward() -> bool:
    """Whether a backward pass is the formula's: to be differentiated again, or
    seen by a dispatch mode."""
    return torch.is_grad_enabled() or torch._C._len_torch_dispatch_stack() > 0


def gradients_of(plain, inputs, needed, grad):
    """The gradients, with a graph of their own where that is wanted: the plain
    formula is run again and differentiated.  It is run on aliases, so
    that each gradient stops at its own input where inputs depend on each other
    or are the same tensor: autograd goes on from there by itself."""
    if not any(needed):
        return [None] * len(inputs)
    again = torch.is_grad_enabled()
    with torch.enable_grad():
        inputs = [None if t is None else t.view_as(t) for t in inputs]
        wanted = [t for t, need in zip(inputs, needed) if need]
        found = iter(torch.autograd.grad(plain(*inputs), wanted, grad, create_graph=again))
        return [next(found) if need else None for need in needed]
