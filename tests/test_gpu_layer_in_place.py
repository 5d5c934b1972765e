"""The layer operators' outputs in the memory of their inputs, where include/helix/helix_layer.h allows it: the same bits
as in memory of their own. Through the C entry points, as the bindings allocate their outputs."""
import pytest
import torch

from helix_amd import abi
from helix_amd.layer import IO_DTYPES, ptr, run, run_with_scratch, scratch
from helix_amd.norm import fp8_rows, rms_norm, rms_norm_backward, rms_norm_fp8
from helix_amd.recurrence import gated_scan

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def stream():
    return torch.cuda.current_stream().cuda_stream


def scan(g, v, h0, h, last):
    S, L, D = g.shape

    def pack(buf, nbytes):
        return abi.GATED_SCAN_STRUCT.pack(S, L, D, IO_DTYPES[g.dtype], ptr(g), ptr(v), ptr(h0), ptr(h), ptr(last), buf, nbytes,
                                          *g.stride()[:2], *v.stride()[:2], *h.stride()[:2])

    L_ = abi.lib()
    run_with_scratch(L_.helix_gated_scan_encode, L_.helix_gated_scan_scratch_size, 0, stream(), None, pack)


# 256 tokens a chunk (above 128), eight chunks a group; few tokens go through a thread.
@pytest.mark.parametrize("L", [0, 1, 16, 100, 256, 257, 512, 1500, 2048, 2049, 10240])
@pytest.mark.parametrize("S,D", [(1, 64), (3, 1000), (40, 130)])
def test_last_in_place_of_h0(gpu, S, D, L):
    g, v, h0 = (2 + normal(S, L, D, seed=1)).bfloat16(), normal(S, L, D, seed=2, dtype=torch.bfloat16), normal(S, D, seed=3)
    want, last = gated_scan(g, v, h0)
    h, state = torch.empty_like(want), h0.clone()
    scan(g, v, state, h, state)
    assert torch.equal(h, want) and torch.equal(state, last)
    # A state that is handed on, sequence by sequence: each call reads what the one before left there.
    scan(g, v, state, h, state)
    again, end = gated_scan(g, v, last)
    assert torch.equal(h, again) and torch.equal(state, end)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [1, 100, 700, 3000])
@pytest.mark.parametrize("D", [64, 201])
def test_h_in_place_of_g_or_v(gpu, L, D, dtype):
    row = normal(2, L, 2 * D + 3, seed=4, dtype=dtype)
    want, last = gated_scan(row[..., :D], row[..., D:2 * D])
    for place in (0, D):
        both = row.clone()
        g, v, end = both[..., :D], both[..., D:2 * D], torch.empty_like(last)
        scan(g, v, None, both[..., place:place + D], end)
        assert torch.equal(both[..., place:place + D], want) and torch.equal(end, last)
        assert torch.equal(both[..., 2 * D:], row[..., 2 * D:])


def norm(x, w, r, h, y=None, q=None, scale=None, rstd=None):
    rows, dim = x.shape
    stride = [0 if t is None else t.stride(0) for t in (x, r, h, y, q, scale)]
    run(abi.lib().helix_norm_encode, 0, stream(),
        abi.NORM_STRUCT.pack(rows, dim, IO_DTYPES[x.dtype], IO_DTYPES[w.dtype], 1e-5, ptr(x), ptr(r), ptr(w), ptr(h), ptr(y), ptr(q),
                             ptr(scale), ptr(rstd), *stride))


# A wave's row, a workgroup's, one that is read twice; even and odd ends.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", [(2000, 256), (1500, 1001), (5, 2048), (7, 5183), (3, 20001)])
def test_h_in_place_of_x_or_residual(gpu, rows, dim, dtype):
    wide = normal(rows, 2 * dim + 1, seed=5, dtype=dtype)
    w = 1 + 0.2 * normal(dim, seed=6)
    y0, h0, rstd0 = rms_norm(wide[:, :dim], w, wide[:, dim + 1:])
    q0, s0, _ = rms_norm_fp8(wide[:, :dim], w, wide[:, dim + 1:])
    for place in (slice(0, dim), slice(dim + 1, 2 * dim + 1)):
        both = wide.clone()
        y, rstd = torch.empty_like(y0), torch.empty_like(rstd0)
        norm(both[:, :dim], w, both[:, dim + 1:], both[:, place], y=y, rstd=rstd)
        assert torch.equal(y, y0) and torch.equal(both[:, place], h0) and torch.equal(rstd, rstd0)
        both = wide.clone()
        q, s = fp8_rows((rows, dim), "cuda")
        norm(both[:, :dim], w, both[:, dim + 1:], both[:, place], q=q, scale=s)
        assert torch.equal(q.float(), q0.float()) and torch.equal(s.float(), s0.float()) and torch.equal(both[:, place], h0)
        assert torch.equal(both[:, dim], wide[:, dim])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", [(2000, 256), (1500, 1001), (5, 2048), (700, 5183), (3, 20001)])
def test_dx_in_place_of_dy_or_dh(gpu, rows, dim, dtype):
    wide = normal(rows, 3 * dim + 1, seed=7, dtype=dtype)
    w = 1 + 0.2 * normal(dim, seed=8)
    h = wide[:, 2 * dim + 1:]
    _, _, rstd = rms_norm(h, w)
    dx0, dw0 = rms_norm_backward(wide[:, :dim], h, w, rstd, wide[:, dim:2 * dim])
    lib = abi.lib()
    for place in (slice(0, dim), slice(dim, 2 * dim)):
        all3, dw = wide.clone(), torch.empty_like(dw0)
        dy, dh, dx, h3 = all3[:, :dim], all3[:, dim:2 * dim], all3[:, place], all3[:, 2 * dim + 1:]

        def pack(buf, nbytes):
            return abi.NORM_BACKWARD_STRUCT.pack(rows, dim, IO_DTYPES[dtype], IO_DTYPES[w.dtype], 0, ptr(dy), ptr(h3), ptr(w), ptr(rstd),
                                                 ptr(dh), ptr(dx), ptr(dw), buf, nbytes, *[3 * dim + 1] * 4)

        need = lib.helix_norm_backward_scratch_size(pack(0, 0))
        run(lib.helix_norm_backward_encode, 0, stream(), pack(ptr(scratch(0, stream(), None, need)), need))
        assert torch.equal(dx, dx0) and torch.equal(dw, dw0)
        assert torch.equal(all3[:, 2 * dim:], wide[:, 2 * dim:])
