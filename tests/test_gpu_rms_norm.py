"""helix_amd.norm on the GPU against the 64-bit forms of layer_oracle.py."""
import pytest
import torch

import layer_oracle as lo
from helix_amd.abi import HelixError
from helix_amd.norm import quantize_fp8, rms_norm, rms_norm_backward, rms_norm_fp8

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
# One channel, less than a wave, ragged and whole blocks, odd widths, wide rows.
DIMS = [1, 7, 64, 127, 128, 130, 384, 1000, 2048, 2560, 4097, 5184, 8192, 16384, 20000, 70001]


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def check_norm(x, w, r, eps=1e-5):
    dim = x.shape[-1]
    want, h64, r64 = lo.norm(x, w, r, eps)
    y, h, rstd = rms_norm(x, w, r, eps=eps)
    lo.within(y, want, lo.norm_bound(want, dim, x.dtype), "y")
    lo.within(rstd, r64, r64 * lo.E * (dim / 64 + 24), "rstd")
    q, scale, h2 = rms_norm_fp8(x, w, r, eps=eps)
    lo.check_fp8(q, scale, want, dim)
    if r is None:
        assert h is x and h2 is x
    else:
        lo.within(h, h64, h64.abs() * (lo.E + lo.U[x.dtype]) + lo.TINY[x.dtype], "h")
        assert torch.equal(h, h2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_norm(gpu, dim, dtype):
    rows = 5 if dim < 20000 else 2
    x, r = 3 * normal(rows, dim, seed=1, dtype=dtype), normal(rows, dim, seed=2, dtype=dtype)
    w = 1 + 0.3 * normal(dim, seed=3)
    check_norm(x, w, r)
    check_norm(x, w.to(dtype), None)


@pytest.mark.parametrize("rows", [1, 2, 3, 63, 257, 4099])
@pytest.mark.parametrize("dim,dtype", [(640, torch.bfloat16), (331, torch.float16), (1023, torch.bfloat16), (1025, torch.float32)])
def test_norm_rows(gpu, rows, dim, dtype):
    check_norm(normal(rows, dim, seed=4, dtype=dtype), 1 + normal(dim, seed=5), None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [96, 1000, 2048, 20000])
def test_norm_strided_and_unaligned(gpu, dim, dtype):
    # Column ranges of wider rows, from a column that no wide load may start at; rows broadcast.
    wide = normal(6, 2 * dim + 5, seed=6, dtype=dtype)
    w = 1 + 0.1 * normal(dim + 1, seed=7)[1:]
    check_norm(wide[:, 3:3 + dim], w, wide[:, dim + 5:])
    check_norm(wide[::2, :dim], w, None)
    check_norm(wide[:1, 1:1 + dim].expand(4, dim), w, wide[:4, 8:8 + dim])
    lead = normal(2, 3, dim, seed=8, dtype=dtype)
    check_norm(lead, w, lead.flip(0))


def test_rows_far_apart(gpu):
    far = torch.empty(3, (1 << 30) + (1 << 29) + 8, device="cuda", dtype=torch.bfloat16)
    x = far[:, :1000]
    x.copy_(normal(3, 1000, seed=80))
    w = 1 + 0.1 * normal(1000, seed=81)
    check_norm(x, w, x)
    _, _, rstd = rms_norm(x, w)
    check_backward(x, x, w, rstd, x)


def test_norm_values(gpu):
    # A zero row, a row of subnormal squares, large values, one lone value, the sum cancelling to zero.
    x = normal(6, 300, seed=9)
    x[0] = 0
    x[1] *= 1e-25
    x[2] *= 1e15
    x[3] = 0
    x[3, 299] = 5
    r = normal(6, 300, seed=10) * 0
    r[4] = -x[4]
    check_norm(x, 1 + normal(300, seed=11), r)
    y, _, rstd = rms_norm(x[:1], torch.ones(300, device="cuda"), eps=0.0)
    assert torch.isinf(rstd).all() and torch.isnan(y).all()   # 0 / 0 by the formula


def test_nan_stays_in_its_row_and_block(gpu):
    x = normal(3, 512, seed=12)
    clean_q, clean_s = quantize_fp8(x)
    x[1, 200] = float("nan")
    y, _, rstd = rms_norm(x, torch.ones(512, device="cuda"))
    assert torch.isnan(y[1]).all() and torch.isnan(rstd[1]) and torch.isfinite(y[[0, 2]]).all()
    q, s = quantize_fp8(x)
    assert torch.isnan(q.float()[1, 200])
    same = torch.ones(3, 512, dtype=torch.bool, device="cuda")
    same[1, 200] = False
    top = clean_q.float()[1, 128:256].abs().argmax()
    if int(top) != 72:
        assert torch.equal(q.float()[same], clean_q.float()[same]) and torch.equal(s.float(), clean_s.float())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 100, 128, 2048, 4097, 20000])
def test_quantize(gpu, dim, dtype):
    x = normal(7, dim, seed=13, dtype=dtype) * torch.exp(2 * normal(dim, seed=14)).to(dtype)
    x[0] = 0
    x[1, :] = 1e-4 if dtype == torch.float16 else 1e-38
    q, scale = quantize_fp8(x)
    lo.check_fp8(q, scale, lo.f64(x), dim)
    if dim >= 128:   # exact borders: 448 stays, anything above doubles the scale
        x = torch.zeros(3, 128, device="cuda")
        x[0, 5], x[1, 6], x[2, 7] = 448.0, 448.0 + 2.0 ** -15, 449.0
        _, s = quantize_fp8(x)
        assert s.float().flatten().tolist() == [1.0, 2.0, 2.0]


def check_backward(dy, h, w, rstd, dh):
    dx64, dw64 = lo.norm_backward(dy, h, w, rstd, dh)
    bx, bw = lo.norm_backward_bound(dy, h, w, rstd, dh, dx64)
    dx, dw = rms_norm_backward(dy, h, w, rstd, dh)
    lo.within(dx, dx64, bx, "dx")
    lo.within(dw, dw64, bw, "dweight")
    dx2, dw2 = rms_norm_backward(dy, h, w, rstd, dh)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_backward(gpu, dim, dtype):
    for rows in (1, 5, 70):
        if rows * dim > 400000:
            continue
        dy, h, dh = (normal(rows, dim, seed=s, dtype=dtype) for s in (20, 21, 22))
        w = 1 + 0.3 * normal(dim, seed=23)
        _, _, rstd = rms_norm(h, w)
        check_backward(dy, h, w, rstd, dh)
        check_backward(dy, h, w.to(dtype), rstd, None)


@pytest.mark.parametrize("rows,dim", [(3001, 96), (513, 1001), (20000, 40), (1500, 333), (700, 4099),
                                      (2100, 2053), (130, 8191)])
def test_backward_many_rows_strided(gpu, rows, dim):
    wide = normal(rows, 3 * dim + 7, seed=24, dtype=torch.bfloat16)
    w = 1 + 0.3 * normal(dim, seed=25)
    h = wide[:, 1:1 + dim]
    _, _, rstd = rms_norm(h, w)
    check_backward(wide[:, dim + 2:2 * dim + 2], h, w, rstd, wide[:, 2 * dim + 7:])


def test_backward_against_differences(gpu):
    # Central differences of the 64-bit forward in random directions: L = sum(cy y) + sum(ch h).
    rows, dim, eps = 6, 150, 1e-5
    x, w = normal(rows, dim, seed=30), 1 + 0.3 * normal(dim, seed=31)
    cy, ch = normal(rows, dim, seed=32), normal(rows, dim, seed=33)
    _, h, rstd = rms_norm(x, w, torch.zeros_like(x), eps=eps)
    dx, dw = rms_norm_backward(cy, h, w, rstd, ch)

    def loss(x, w):
        y, h, _ = lo.norm(x, w, None, eps)
        return float((lo.f64(cy) * y).sum() + (lo.f64(ch) * h).sum())

    for seed in range(4):
        px, pw = lo.f64(normal(rows, dim, seed=40 + seed)), lo.f64(normal(dim, seed=50 + seed))
        d = 1e-5
        x64, w64 = lo.f64(x), lo.f64(w)
        num = (loss(x64 + d * px, w64 + d * pw) - loss(x64 - d * px, w64 - d * pw)) / (2 * d)
        ana = float((lo.f64(dx) * px).sum() + (lo.f64(dw) * pw).sum())
        # fp32 gradients: 1e-6 of the terms' magnitudes; differences: d^2 times a third derivative.
        size = float((lo.f64(dx) * px).abs().sum() + (lo.f64(dw) * pw).abs().sum())
        assert abs(num - ana) <= 1e-6 * size


def test_no_rows(gpu):
    e = torch.empty(0, 256, device="cuda")
    w = torch.ones(256, device="cuda")
    y, h, rstd = rms_norm(e, w)
    assert y.shape == (0, 256) and rstd.shape == (0,)
    q, scale, _ = rms_norm_fp8(e, w)
    assert q.shape == (0, 256) and scale.shape == (0, 2)
    dx, dw = rms_norm_backward(e, e, w, torch.empty(0, device="cuda"))
    assert dx.shape == (0, 256) and (dw == 0).all()


def test_other_stream_and_graph(gpu):
    x, r = normal(300, 2560, seed=60, dtype=torch.bfloat16), normal(300, 2560, seed=61, dtype=torch.bfloat16)
    w, dy = 1 + 0.2 * normal(2560, seed=62), normal(300, 2560, seed=63, dtype=torch.bfloat16)

    def step(stream=None):
        y, h, rstd = rms_norm(x, w, r, stream=stream)
        q, scale, _ = rms_norm_fp8(x, w, r, stream=stream)
        return (y, h, rstd, q.float(), scale.float(), *rms_norm_backward(dy, h, w, rstd, h, stream=stream))

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(3):
        x.copy_(normal(300, 2560, seed=70 + k))
        graph.replay()
        torch.cuda.synchronize()
        again = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(again, step()))


def test_refusals(gpu):
    x, w = normal(4, 64), torch.ones(64, device="cuda")
    for bad in (dict(x=x.double()), dict(x=x.cpu()), dict(weight=w[:63]), dict(weight=w.half()),
                dict(residual=x[:3]), dict(residual=x.half()), dict(x=normal(64, 4).t()),
                dict(x=normal(4, 6, 64)[:, ::2].transpose(0, 1), weight=w)):
        with pytest.raises(ValueError):
            rms_norm(**{"x": x, "weight": w, "residual": None, **bad})
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(HelixError):
            rms_norm(x, w, eps=eps)
    _, _, rstd = rms_norm(x, w)
    for bad in (dict(dy=x.half()), dict(rstd=rstd[:3]), dict(rstd=rstd.half()), dict(dh=x[:, :60]), dict(weight=w[1:])):
        with pytest.raises(ValueError):
            rms_norm_backward(**{"dy": x, "h": x, "weight": w, "rstd": rstd, **bad})
