"""What the layer operators' bindings (helix_amd.norm, helix_amd.matmul, helix_amd.recurrence) share: checks of
tensors, streams, scratch and errors. The arithmetic runs in the HIP kernels of libhelix.so
(include/helix/helix_layer.h)."""
from __future__ import annotations

import contextlib
import struct

import torch

from .abi import HelixError
from .desc import HELIX_BF16, HELIX_ERR_SCRATCH_TOO_SMALL, HELIX_F16, HELIX_F32, HELIX_OK
from .scan import _capturing, _contexts, _scratch_for, _under, context

IO_DTYPES = {torch.float32: HELIX_F32, torch.bfloat16: HELIX_BF16, torch.float16: HELIX_F16}
FP8 = torch.float8_e4m3fn
FP8_SCALE = torch.float8_e8m0fnu
# HELIX_FP8_BLOCK: elements of a row that share a scale
FP8_BLOCK = 128


def device_index(op: str, t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise ValueError(f"{op} runs on a HIP device; got {t.device}")
    return t.get_device()


def io_code(name: str, t: torch.Tensor) -> int:
    code = IO_DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16; got {t.dtype}")
    return code


def expect(name: str, t: torch.Tensor, dtype: torch.dtype, shape, like: torch.Tensor) -> None:
    if t.dtype != dtype or t.get_device() != like.get_device():
        raise ValueError(f"{name} must be {dtype} on {like.device}; got {t.dtype} on {t.device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}; got {tuple(t.shape)}")


def row_stride(name: str, t: torch.Tensor) -> int:
    """The one stride of the rows of t [..., dim], whose leading dimensions have to collapse into one."""
    if t.is_contiguous():
        return t.shape[-1]
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    ld = None     # stride of the rows so far, from the inside out
    span = 0      # stride that the next dimension has to have
    for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if ld is None:
            ld = s
        elif s != span:
            raise ValueError(f"{name}: the leading dimensions must collapse into rows of one stride")
        span = s * n
    return t.shape[-1] if ld is None else ld


def empty(shape, dtype: torch.dtype, device) -> torch.Tensor:
    """Uninitialised. (Sizes one by one spare half of what torch.empty takes for a torch.Size.)"""
    return torch.empty(*shape, dtype=dtype, device=device) if shape else torch.empty((), dtype=dtype, device=device)


def rows_like(t: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    """Uninitialised and contiguous, of t's shape and, unless another is given, type."""
    if t.is_contiguous():
        return torch.empty_like(t, dtype=dtype)
    return empty(t.shape, dtype or t.dtype, t.device)


def stream_handle(index: int, stream) -> int:
    return stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(index)


_here = contextlib.nullcontext()


def under(index: int, stream):
    """The context that outputs are allocated in, so that their memory is the stream's own."""
    return _here if stream is None else _under(index, stream.cuda_stream, stream)


def scratch(index: int, st: int, stream, nbytes: int) -> torch.Tensor | None:
    """Scratch of the calling thread for the stream; work under capture gets memory of the graph's own."""
    if not nbytes:
        return None
    if torch.cuda.is_current_stream_capturing() if stream is None else _capturing(index, st, stream):
        with _under(index, st, stream):
            return torch.empty(nbytes, dtype=torch.uint8, device=f"cuda:{index}")
    return _scratch_for(index, st, nbytes, stream)


def packed(pack, *fields) -> bytes:
    """pack(*fields), an argument struct of helix_amd.abi; what its fields cannot hold is refused."""
    try:
        return pack(*fields)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"a size, a stride or eps is out of range: {e}") from None


def run(fn, index: int, st: int, args: bytes) -> None:
    ctx = _contexts.get(index) or context(index)
    rc = fn(ctx.handle, st, args)
    if rc != HELIX_OK:
        raise HelixError(rc, ctx.last_error())


def run_with_scratch(fn, size, index: int, st: int, stream, pack) -> None:
    """run for an operator that may want scratch: pack(address, bytes) gives its arguments, size(arguments) the bytes.
    It is asked for them once the call has been refused without (nothing is enqueued then): the small calls, whose time
    on the host counts, want none."""
    ctx = _contexts.get(index) or context(index)
    args = packed(pack, 0, 0)
    rc = fn(ctx.handle, st, args)
    if rc == HELIX_ERR_SCRATCH_TOO_SMALL:
        need = size(args)
        buf = scratch(index, st, stream, need)
        rc = fn(ctx.handle, st, pack(ptr(buf), need))
    if rc != HELIX_OK:
        raise HelixError(rc, ctx.last_error())


def ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()
