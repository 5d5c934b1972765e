"""Product of two 8-bit matrices with a scale for each block of 128 along the sum (include/helix/helix_layer.h)."""
from __future__ import annotations

import torch

from . import abi
from .layer import (FP8, FP8_BLOCK, FP8_SCALE, IO_DTYPES, device_index, expect, row_stride, run_with_scratch,
                    stream_handle, under)


def matmul_fp8(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, *,
               out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
               stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """a [..., k] times b [n, k] transposed: [..., n] in out_dtype (float32, bfloat16 or float16), or into `out`.

    Sums are float32. float32 results are sums of exact products; for the 16-bit ones, rounded once, the matrix
    instruction cuts each of eight neighbouring products at 2^-13 of the largest of them (2e-5 of a result on ordinary
    operands, and no less where products cancel: include/helix/helix_layer.h).

    a and b are float8_e4m3fn, a_scale [..., ceil(k / 128)] and b_scale [n, ceil(k / 128)] float8_e8m0fnu, as
    rms_norm_fp8 and quantize_fp8 leave them. Rows of a and b start at multiples of 16 bytes; k is any length."""
    index = device_index("matmul_fp8", a)
    if a.dim() < 1 or b.dim() != 2 or a.shape[-1] < 1:
        raise ValueError("a must be [..., k] and b [n, k], k at least 1")
    k = a.shape[-1]
    n = b.shape[0]
    blocks = -(-k // FP8_BLOCK)
    lead = a.shape[:-1]
    expect("a", a, FP8, a.shape, a)
    expect("b", b, FP8, (n, k), a)
    expect("a_scale", a_scale, FP8_SCALE, (*lead, blocks), a)
    expect("b_scale", b_scale, FP8_SCALE, (n, blocks), a)
    if out is None:
        if out_dtype not in IO_DTYPES:
            raise ValueError(f"out_dtype must be float32, bfloat16 or float16; got {out_dtype}")
        with under(index, stream):
            out = torch.empty(*lead, n, dtype=out_dtype, device=a.device)
        ld_c = n
    else:
        if out.dtype not in IO_DTYPES:
            raise ValueError(f"out must be float32, bfloat16 or float16; got {out.dtype}")
        expect("out", out, out.dtype, (*lead, n), a)
        ld_c = row_stride("out", out)
    st = stream_handle(index, stream)
    dims = (a.numel() // k, n, k, IO_DTYPES[out.dtype], a.data_ptr(), a_scale.data_ptr(), b.data_ptr(),
            b_scale.data_ptr(), out.data_ptr())
    strides = (row_stride("a", a), row_stride("a_scale", a_scale), row_stride("b", b), row_stride("b_scale", b_scale), ld_c)

    def pack(buf, nbytes):
        return abi.MATMUL_FP8_STRUCT.pack(*dims, buf, nbytes, *strides)

    lib = abi.lib()
    run_with_scratch(lib.helix_matmul_fp8_encode, lib.helix_matmul_fp8_scratch_size, index, st, stream, pack)
    return out
