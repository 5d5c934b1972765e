"""The layer operators' C ABI without a GPU: exported symbols, struct layouts, checks of arguments; and the 64-bit
forms that the GPU tests compare with, against each other."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import layer_oracle as lo
from helix_amd import abi
from helix_amd.desc import (HELIX_ERR_INVALID_ARG, HELIX_ERR_NO_DEVICE, HELIX_ERR_SCRATCH_TOO_SMALL,
                            HELIX_ERR_UNSUPPORTED_SHAPE, HELIX_OK)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"helix_norm_args": abi.NORM_STRUCT, "helix_norm_backward_args": abi.NORM_BACKWARD_STRUCT,
           "helix_matmul_fp8_args": abi.MATMUL_FP8_STRUCT, "helix_gated_scan_args": abi.GATED_SCAN_STRUCT,
           "helix_gated_scan_backward_args": abi.GATED_SCAN_BACKWARD_STRUCT}


@pytest.fixture(scope="module")
def host():
    c = abi.Context(host_only=True)
    yield c
    c.close()


def header():
    text = open(os.path.join(ROOT, "include", "helix", "helix_layer.h")).read()
    return re.sub(r"/\*.*?\*/", "", text, flags=re.S)


def test_every_declared_symbol_is_exported():
    declared = set(re.findall(r"\b(helix_[a-z_0-9]+)\s*\(", header()))
    assert declared == set(abi.LAYER_SYMBOLS)
    L = abi.lib()
    assert all(hasattr(L, name) for name in declared)


def test_packed_arguments_match_the_header(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text("#include <stdio.h>\n#include \"helix/helix_layer.h\"\nint main(void) {\n" +
                   "".join(f'printf("{n} %zu\\n", sizeof({n}));\n' for n in STRUCTS) + "return 0;\n}\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    assert {n: int(v) for n, v in out.items()} == {n: s.size for n, s in STRUCTS.items()}


def call(host, name, args):
    return int(getattr(abi.lib(), name)(host.handle, None, args))


P = 1 << 12   # an address that nothing reads: every check is made before a launch


def norm_args(rows=4, dim=200, io=2, w=0, eps=1e-5, x=P, r=0, weight=P, h=0, y=P, q=0, scale=0, rstd=P, ld=256):
    return abi.NORM_STRUCT.pack(rows, dim, io, w, eps, x, r, weight, h, y, q, scale, rstd, *[ld] * 6)


@pytest.mark.parametrize("change,status,word", [
    (dict(), HELIX_ERR_NO_DEVICE, "no device"),
    (dict(rows=0), HELIX_OK, ""),
    (dict(rows=-1), HELIX_ERR_UNSUPPORTED_SHAPE, "rows"),
    (dict(dim=0), HELIX_ERR_UNSUPPORTED_SHAPE, "dim"),
    (dict(dim=(1 << 20) + 1), HELIX_ERR_UNSUPPORTED_SHAPE, "dim"),
    (dict(io=3), HELIX_ERR_INVALID_ARG, "io_dtype"),
    (dict(w=1), HELIX_ERR_INVALID_ARG, "weight_dtype"),
    (dict(eps=float("nan")), HELIX_ERR_INVALID_ARG, "eps"),
    (dict(x=0), HELIX_ERR_INVALID_ARG, "x is NULL"),
    (dict(x=P + 1), HELIX_ERR_INVALID_ARG, "aligned"),
    (dict(weight=0), HELIX_ERR_INVALID_ARG, "weight"),
    (dict(weight=P + 2), HELIX_ERR_INVALID_ARG, "aligned"),
    (dict(q=P, scale=P), HELIX_ERR_INVALID_ARG, "exactly one"),
    (dict(y=0), HELIX_ERR_INVALID_ARG, "exactly one"),
    (dict(y=0, q=P), HELIX_ERR_INVALID_ARG, "scale"),
    (dict(ld=199), HELIX_ERR_INVALID_ARG, "overlap"),
    (dict(ld=-256), HELIX_ERR_INVALID_ARG, "stride"),
    (dict(rstd=P + 2), HELIX_ERR_INVALID_ARG, "rstd"),
    (dict(rows=1 << 34), HELIX_ERR_INVALID_ARG, "grid"),
])
def test_norm_checks(host, change, status, word):
    assert call(host, "helix_norm_encode", norm_args(**change)) == status
    if status != HELIX_OK:
        assert word in host.last_error()


def test_quantize_checks(host):
    good = dict(weight=0, rstd=0, y=0, q=P, scale=P)
    assert call(host, "helix_quantize_fp8_encode", norm_args(**good)) == HELIX_ERR_NO_DEVICE
    for bad in (dict(weight=P), dict(rstd=P), dict(y=P), dict(q=0), dict(scale=0)):
        assert call(host, "helix_quantize_fp8_encode", norm_args(**{**good, **bad})) == HELIX_ERR_INVALID_ARG


def bwd_args(rows=100, dim=200, io=2, w=0, res=0, dy=P, h=P, weight=P, rstd=P, dh=0, dx=P, dw=P, scratch=P,
             nbytes=1 << 30, ld=256):
    return abi.NORM_BACKWARD_STRUCT.pack(rows, dim, io, w, res, dy, h, weight, rstd, dh, dx, dw, scratch, nbytes, *[ld] * 4)


@pytest.mark.parametrize("change,status", [
    (dict(), HELIX_ERR_NO_DEVICE), (dict(rows=0, dw=0), HELIX_OK), (dict(rows=-1), HELIX_ERR_UNSUPPORTED_SHAPE),
    (dict(dim=0), HELIX_ERR_UNSUPPORTED_SHAPE), (dict(io=-1), HELIX_ERR_INVALID_ARG), (dict(w=1), HELIX_ERR_INVALID_ARG),
    (dict(res=1), HELIX_ERR_INVALID_ARG), (dict(dy=0), HELIX_ERR_INVALID_ARG), (dict(rstd=0), HELIX_ERR_INVALID_ARG),
    (dict(dx=0), HELIX_ERR_INVALID_ARG), (dict(ld=100), HELIX_ERR_INVALID_ARG), (dict(dw=P + 1), HELIX_ERR_INVALID_ARG),
    (dict(scratch=0), HELIX_ERR_SCRATCH_TOO_SMALL), (dict(nbytes=16), HELIX_ERR_SCRATCH_TOO_SMALL),
    (dict(scratch=P + 4), HELIX_ERR_INVALID_ARG), (dict(dw=0, scratch=0, nbytes=0), HELIX_ERR_NO_DEVICE),
])
def test_norm_backward_checks(host, change, status):
    assert call(host, "helix_norm_backward_encode", bwd_args(**change)) == status


def mm_args(m=4, n=8, k=300, out=2, a=P, sa=P, b=P, sb=P, c=P, scratch=P, nbytes=1 << 20, lda=304, ldsa=3,
            ldb=304, ldsb=3, ldc=8):
    return abi.MATMUL_FP8_STRUCT.pack(m, n, k, out, a, sa, b, sb, c, scratch, nbytes, lda, ldsa, ldb, ldsb, ldc)


@pytest.mark.parametrize("change,status", [
    (dict(), HELIX_ERR_NO_DEVICE), (dict(m=0), HELIX_OK), (dict(n=0), HELIX_OK), (dict(m=-1), HELIX_ERR_UNSUPPORTED_SHAPE),
    (dict(k=0), HELIX_ERR_UNSUPPORTED_SHAPE), (dict(k=(1 << 20) + 1), HELIX_ERR_UNSUPPORTED_SHAPE),
    (dict(out=3), HELIX_ERR_INVALID_ARG), (dict(a=0), HELIX_ERR_INVALID_ARG), (dict(a=P + 8), HELIX_ERR_INVALID_ARG),
    (dict(b=P + 1), HELIX_ERR_INVALID_ARG), (dict(sa=0), HELIX_ERR_INVALID_ARG), (dict(lda=312), HELIX_ERR_INVALID_ARG),
    (dict(m=1000, k=600, lda=608, ldb=608, ldsa=5, nbytes=10), HELIX_ERR_SCRATCH_TOO_SMALL),
    (dict(m=1000, k=600, lda=608, ldb=608, ldsa=5, scratch=0), HELIX_ERR_SCRATCH_TOO_SMALL),
    (dict(m=1000, k=600, lda=608, ldb=608, ldsa=8, ldsb=8, scratch=0, nbytes=0), HELIX_ERR_NO_DEVICE),
    (dict(ldb=-304), HELIX_ERR_INVALID_ARG), (dict(ldc=7), HELIX_ERR_INVALID_ARG), (dict(c=P + 1), HELIX_ERR_INVALID_ARG),
])
def test_matmul_checks(host, change, status):
    assert call(host, "helix_matmul_fp8_encode", mm_args(**change)) == status


def scan_args(S=2, L=2000, D=64, io=2, g=P, v=P, h0=0, h=P, last=P, scratch=P, nbytes=1 << 30, seq=128000, tok=64):
    return abi.GATED_SCAN_STRUCT.pack(S, L, D, io, g, v, h0, h, last, scratch, nbytes, *[seq, tok] * 3)


def scan_bwd_args(S=2, L=2000, D=64, io=2, dh=P, g=P, v=P, h=P, h0=0, dl=0, dg=P, dv=P, dh0=P, scratch=P, nbytes=1 << 30,
                  seq=128000, tok=64):
    return abi.GATED_SCAN_BACKWARD_STRUCT.pack(S, L, D, io, dh, g, v, h, h0, dl, dg, dv, dh0, scratch, nbytes,
                                               *[seq, tok] * 6)


@pytest.mark.parametrize("make,name", [(scan_args, "helix_gated_scan_encode"),
                                       (scan_bwd_args, "helix_gated_scan_backward_encode")])
@pytest.mark.parametrize("change,status", [
    (dict(), HELIX_ERR_NO_DEVICE), (dict(S=0), HELIX_OK), (dict(D=0), HELIX_OK), (dict(L=-1), HELIX_ERR_UNSUPPORTED_SHAPE),
    (dict(io=9), HELIX_ERR_INVALID_ARG), (dict(g=0), HELIX_ERR_INVALID_ARG), (dict(v=P + 1), HELIX_ERR_INVALID_ARG),
    (dict(h=0), HELIX_ERR_INVALID_ARG), (dict(tok=63), HELIX_ERR_INVALID_ARG), (dict(tok=-64), HELIX_ERR_INVALID_ARG),
    (dict(seq=-1), HELIX_ERR_INVALID_ARG), (dict(seq=0), HELIX_ERR_INVALID_ARG), (dict(h0=P + 2), HELIX_ERR_INVALID_ARG),
])
def test_scan_checks(host, make, name, change, status):
    assert call(host, name, make(**change)) == status


def test_null_arguments(host):
    for name in abi.LAYER_SYMBOLS:
        fn = getattr(abi.lib(), name)
        if name.endswith("_size"):
            assert fn(None) == 0
        else:
            assert fn(host.handle, None, None) == HELIX_ERR_INVALID_ARG
            assert fn(None, None, bytes(256)) == HELIX_ERR_INVALID_ARG


# ---- the 64-bit forms ---------------------------------------------------------

def test_oracle_gradients_by_differentiation():
    torch.manual_seed(0)
    g, v = (torch.randn(2, 7, 3, dtype=torch.float64, requires_grad=True) for _ in range(2))
    h0 = torch.randn(2, 3, dtype=torch.float64, requires_grad=True)
    hs, s = [], h0
    for t in range(7):
        s = torch.sigmoid(g[:, t]) * s + (1 - torch.sigmoid(g[:, t])) * v[:, t]
        hs.append(s)
    h = torch.stack(hs, 1)
    assert torch.allclose(lo.scan(g, v, h0)[0], h, rtol=1e-14, atol=1e-14)
    dh, dl = torch.randn(2, 7, 3, dtype=torch.float64), torch.randn(2, 3, dtype=torch.float64)
    want = torch.autograd.grad((h * dh).sum() + (s * dl).sum(), (g, v, h0))
    for a, b in zip(lo.scan_backward(dh, g, v, h, h0, dl), want):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-13)
    x, w = torch.randn(5, 11, dtype=torch.float64, requires_grad=True), torch.randn(11, dtype=torch.float64, requires_grad=True)
    rstd = (x.square().mean(-1) + 1e-5).rsqrt()
    y = x * rstd[:, None] * w
    dy, dh = torch.randn(5, 11, dtype=torch.float64), torch.randn(5, 11, dtype=torch.float64)
    want = torch.autograd.grad((y * dy).sum() + (x * dh).sum(), (x, w))
    for a, b in zip(lo.norm_backward(dy, x, w, rstd, dh), want):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-13)


def test_the_checks_see_a_mistake():
    # Planted in the 64-bit side: a block's scale from its neighbour, a row's missing last token, a lost carry.
    torch.manual_seed(1)
    y = torch.randn(3, 256, dtype=torch.float64) * torch.tensor([1.0, 8.0]).repeat_interleave(128)
    s = torch.exp2(torch.ceil(torch.log2(lo.blocks(y).abs().amax(-1) / 448)))
    q = (y / lo.expand(s, 256)).float().to(torch.float8_e4m3fn)
    lo.check_fp8(q, s, y, 256)
    with pytest.raises(AssertionError):
        lo.check_fp8(q, s.flip(1), y, 256)
    g, v, h0 = 2 + torch.randn(1, 50, 4), torch.randn(1, 50, 4), torch.randn(1, 4)
    h, last = lo.scan(g, v, h0)
    bh, bl = lo.scan_bound(g, v, h0, h)
    lo.within(h.float(), h, bh)
    with pytest.raises(AssertionError):
        lo.within(lo.scan(g, v, None)[0].float(), h, bh)
    with pytest.raises(AssertionError):
        lo.within(h[:, -2].float(), last, bl)


# ---- what the compiler cannot see in the tiles' assembly ------------------------

HSACO = os.path.join(ROOT, "helix_amd", "csrc", "_build", "helix_kernels.hsaco")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def _registers(token):
    m = re.match(r"([vas])\[(\d+):(\d+)\]", token)
    if m:
        return {(m.group(1), k) for k in range(int(m.group(2)), int(m.group(3)) + 1)}
    m = re.match(r"([vas])(\d+)$", token)
    return {(m.group(1), int(m.group(2)))} if m else set()


def _missing_waits(lines):
    """Products that read a register a vector instruction wrote less than two wait states before, and loads into LDS
    that read a scalar one wrote less than five before."""
    def operands(line):
        return [t.split(" ")[0] for t in re.split(r",\s*(?![^\[]*\])", line.split(None, 1)[1])] if " " in line else []

    found = []
    for i, line in enumerate(lines):
        if line.startswith("v_mfma_scale"):
            reads, states = set().union(*(_registers(t) for t in operands(line)[1:])), 2
        elif line.startswith("buffer_load") and line.endswith("lds"):
            reads, states = {r for t in operands(line) for r in _registers(t) if r[0] == "s"}, 5
        else:
            continue
        passed = 0
        for before in reversed(lines[max(0, i - 8):i]):
            if before.startswith("v_") and not before.startswith("v_mfma") and operands(before):
                wrote = _registers(operands(before)[0])
                if wrote & reads and passed < states:
                    found.append((before, line))
            m = re.match(r"s_nop (\d+)", before)
            passed += int(m.group(1)) + 1 if m else 1
            if passed >= states:
                break
    return found


def test_missing_waits_are_seen():
    product = "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[8:15], v[16:23], a[0:3], v30, v31 op_sel_hi:[0,0,0]"
    load = "buffer_load_dwordx4 v2, s[4:7], s9 offen lds"
    assert _missing_waits(["v_lshrrev_b32_e32 v30, s2, v30", product])
    assert _missing_waits(["v_mov_b32_e32 v10, v11", "s_mov_b32 s0, 0", product])
    assert not _missing_waits(["v_mov_b32_e32 v10, v11", "s_nop 1", product])
    assert _missing_waits(["v_readlane_b32 s9, v255, 3", "s_add_u32 m0, s1, 0x400", "s_nop 0", load])
    assert not _missing_waits(["v_readlane_b32 s9, v255, 3", "s_mov_b32 m0, s1", "s_nop 4", load])


@pytest.mark.skipif(not (os.path.exists(HSACO) and os.path.exists(OBJDUMP)), reason="needs the built code object and llvm-objdump")
def test_tiles_assembly_waits_for_its_operands():
    out = subprocess.run([OBJDUMP, "-d", HSACO], check=True, capture_output=True, text=True).stdout
    kernels = 0
    for block in re.split(r"\n(?=[0-9a-f]+ <)", out):
        name = re.match(r"[0-9a-f]+ <(\w+)>", block)
        if not name or not re.match(r"helix_matmul_fp8_t\d", name.group(1)):
            continue
        kernels += 1
        lines = [re.sub(r"\s+", " ", ln.split("//")[0]).strip() for ln in block.splitlines()[1:]]
        assert _missing_waits([ln for ln in lines if ln]) == [], name.group(1)
    assert kernels == 7
