"""helix_amd.norm.group_norm on the GPU against the 64-bit forms of group_norm_oracle.py."""
import pytest
import torch

import group_norm_oracle as go
import layer_oracle as lo
from helix_amd import abi
from helix_amd.abi import HelixError
from helix_amd.layer import IO_DTYPES, packed, ptr, run
from helix_amd.norm import group_norm, group_norm_backward, group_norm_fp8, quantize_fp8

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = float("inf")
# (groups, their width): every form of the kernels, whole and cut by the group's end.
GROUPS = [(1, 1), (7, 1), (3, 5), (4, 8), (2, 31), (5, 32), (64, 64), (3, 64), (2, 65), (9, 80), (27, 95), (2, 127),
          (2, 128), (5, 192), (3, 255), (2, 256), (1, 511), (3, 512), (2, 513), (1, 1024), (2, 1025), (1, 2048), (1, 2049),
          (2, 4096), (1, 4097), (1, 8191), (1, 8192)]


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def problem(rows, groups, width, dtype, seed=0, gated=True, biased=True, own_weights=False):
    dim = groups * width
    x = (normal(rows, dim, seed=seed) + 0.5 * normal(dim, seed=seed + 1)).to(dtype)
    wt = dtype if own_weights else torch.float32
    w = (1 + 0.3 * normal(dim, seed=seed + 2)).to(wt)
    b = (0.2 * normal(dim, seed=seed + 3)).to(wt) if biased else None
    return x, w, b, normal(rows, dim, seed=seed + 4, dtype=dtype) if gated else None


def check(x, w, b, gate, groups, kind="silu", eps=1e-5):
    y64, mean64, rstd64, z64 = go.forward(x, w, b, gate, groups, kind, eps)
    by, bm, br = go.forward_bound(x, w, b, gate, groups, kind, eps, y64, mean64, rstd64, z64)
    y, mean, rstd = group_norm(x, w, b, gate, groups=groups, activation=kind, eps=eps)
    lo.within(y, y64, by, "y")
    lo.within(mean, mean64, bm, "mean")
    lo.within(rstd, rstd64, br, "rstd")
    return mean, rstd


def check_backward(dy, x, w, mean, rstd, b, gate, groups, kind="silu"):
    args = (dy, x, w, mean, rstd, b, gate)
    want = go.backward(*args, groups, kind)
    bounds = go.backward_bound(*args, groups, kind, want[0], want[3])
    got = group_norm_backward(*args, groups=groups, activation=kind)
    for name, g, v, c in zip(("dx", "dweight", "dbias", "dgate"), got, want, bounds):
        if g is None:
            assert b is None if name == "dbias" else gate is None
        else:
            lo.within(g, v, c, name)
    again = group_norm_backward(*args, groups=groups, activation=kind)
    assert all(a is None and g is None or torch.equal(a, g) for a, g in zip(again, got))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups,width", GROUPS)
def test_groups(gpu, groups, width, dtype):
    for rows in (1, 6, 67):
        if rows * groups * width > 400000:
            continue
        x, w, b, gate = problem(rows, groups, width, dtype, seed=width, gated=rows != 6, biased=rows != 67,
                                own_weights=rows == 6)
        mean, rstd = check(x, w, b, gate, groups)
        check_backward(normal(*x.shape, seed=9, dtype=dtype), x, w, mean, rstd, b, gate, groups)


@pytest.mark.parametrize("kind", [None, "silu", "sigmoid"])
@pytest.mark.parametrize("gated", [False, True])
def test_activations(gpu, kind, gated):
    x, w, b, gate = problem(33, 6, 80, torch.float32, seed=3, gated=gated)
    if gated:
        gate[0, :4] = torch.tensor([80.0, -80.0, 1e-30, 0.0])
        gate[1] *= 30
    mean, rstd = check(x, w, b, gate, 6, kind)
    check_backward(normal(33, 480, seed=4), x, w, mean, rstd, b, gate, 6, kind)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups,width", [(5, 64), (3, 95), (1, 640), (4, 128), (12, 32), (7, 33)])
def test_strided_rows(gpu, groups, width, dtype):
    dim = groups * width
    wide = normal(70, 3 * dim + 13, seed=5, dtype=dtype)
    x, gate, dy = wide[:, 1:1 + dim], wide[:, dim + 4:2 * dim + 4], wide[:, 2 * dim + 13:]
    w = 1 + 0.1 * normal(dim, seed=6)
    mean, rstd = check(x, w, None, gate, groups)
    check_backward(dy, x, w, mean, rstd, None, gate, groups)


def test_many_rows(gpu):
    x, w, b, gate = problem(20000, 4, 24, torch.bfloat16, seed=7)
    mean, rstd = check(x, w, b, gate, 4)
    check_backward(normal(20000, 96, seed=8, dtype=torch.bfloat16), x, w, mean, rstd, b, gate, 4)
    x, w, b, _ = problem(3000, 1, 700, torch.float16, seed=9, gated=False)
    mean, rstd = check(x, w, b, None, 1)
    check_backward(normal(3000, 700, seed=10, dtype=torch.float16), x, w, mean, rstd, b, None, 1)


def test_far_from_zero(gpu):
    # A mean a thousand times the spread: the variance is of differences. And constant groups: rstd is eps's.
    x, w, b, gate = problem(9, 4, 64, torch.float32, seed=11)
    x = x * 0.01 + 30
    check(x, w, b, gate, 4)
    x = torch.full((3, 256), 7.0, device="cuda")
    y, mean, rstd = group_norm(x, w, b, groups=4, activation=None)
    assert torch.equal(y, b.expand(3, 256)) and (mean == 7).all()
    assert (rstd - 1e-5 ** -0.5).abs().max() < 1e-4


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups,width", [(64, 64), (6, 64), (4, 32), (3, 32), (2, 128), (3, 384), (1, 1024), (1, 2176),
                                          (27, 95), (5, 16), (3, 80), (1, 1), (2, 4096), (1, 129), (80, 192), (8, 2048)])
def test_fp8(gpu, groups, width, dtype):
    x, w, b, gate = problem(5, groups, width, dtype, seed=width, gated=width % 3 != 0, biased=groups != 3)
    dim = groups * width
    y64, mean64, rstd64, z64 = go.forward(x, w, b, gate, groups, "silu", 1e-5)
    off = go.forward_bound(x.float(), w, b, gate, groups, "silu", 1e-5, y64, mean64, rstd64, z64)[0]
    q, scale = group_norm_fp8(x, w, b, gate, groups=groups)
    s = lo.expand(lo.f64(scale.float()), dim)
    got = lo.f64(q.float()) * s
    # e4m3: half of a last place of four bits, or of the least subnormal 2^-9; and y's own error.
    assert ((got - y64).abs() <= (y64.abs() + off) * 2.0 ** -4 + off + 2.0 ** -10 * s).all()
    top, err = lo.blocks(y64).abs().amax(-1), lo.blocks(off).amax(-1)
    sb = lo.f64(scale.float())
    assert (top - err <= 448 * sb).all() and ((224 * sb < top + err) | (sb == 2.0 ** -126)).all()
    # The layout that matmul_fp8 takes, as quantize_fp8 leaves it.
    q2, s2 = quantize_fp8(x)
    assert q.stride() == q2.stride() and scale.stride() == s2.stride()


def test_infinite_and_nan_stay_in_their_group(gpu):
    x, w, b, gate = problem(4, 6, 40, torch.bfloat16, seed=20)
    want, _, _ = group_norm(x, w, b, gate, groups=6)
    bad = x.clone()
    bad[1, 41], bad[2, 239] = INF, float("nan")
    y, mean, rstd = group_norm(bad, w, b, gate, groups=6)
    assert y[1, 40:80].isnan().all() and y[2, 200:].isnan().all()
    y[1, 40:80], y[2, 200:] = want[1, 40:80], want[2, 200:]
    assert torch.equal(y, want)
    dy = normal(4, 240, seed=21, dtype=torch.bfloat16)
    clean = group_norm_backward(dy, x, w, *group_norm(x, w, b, gate, groups=6)[1:], b, gate, groups=6)[0]
    dx = group_norm_backward(dy, bad, w, mean, rstd, b, gate, groups=6)[0]
    assert dx[1, 40:80].isnan().all() and dx[2, 200:].isnan().all()
    dx[1, 40:80], dx[2, 200:] = clean[1, 40:80], clean[2, 200:]
    assert torch.equal(dx, clean)


def test_against_differences(gpu):
    # Central differences of the 64-bit forward in random directions.
    x, w, b, gate = problem(6, 3, 50, torch.float32, seed=30)
    cy = normal(6, 150, seed=31)
    _, mean, rstd = group_norm(x, w, b, gate, groups=3)
    got = group_norm_backward(cy, x, w, mean, rstd, b, gate, groups=3)
    at = [lo.f64(t) for t in (x, w, b, gate)]

    def loss(x, w, b, gate):
        return float((lo.f64(cy) * go.forward(x, w, b, gate, 3, "silu", 1e-5)[0]).sum())

    for seed in range(4):
        way = [lo.f64(normal(*t.shape, seed=40 + 4 * seed + i)) for i, t in enumerate(at)]
        d = 1e-5
        num = (loss(*[t + d * p for t, p in zip(at, way)]) - loss(*[t - d * p for t, p in zip(at, way)])) / (2 * d)
        ana = sum(float((lo.f64(g) * p).sum()) for g, p in zip(got, way))
        size = sum(float((lo.f64(g) * p).abs().sum()) for g, p in zip(got, way))
        assert abs(num - ana) <= 2e-6 * size


def test_no_rows(gpu):
    e, w = torch.empty(0, 96, device="cuda"), torch.ones(96, device="cuda")
    y, mean, rstd = group_norm(e, w, groups=3)
    assert y.shape == (0, 96) and mean.shape == (0, 3) and rstd.shape == (0, 3)
    q, scale = group_norm_fp8(e, w, groups=3)
    assert q.shape == (0, 96) and scale.shape == (0, 1)
    dx, dw, db, dgate = group_norm_backward(e, e, w, mean, rstd, w, e, groups=3)
    assert dx.shape == dgate.shape == (0, 96) and (dw == 0).all() and (db == 0).all()


def test_outputs_in_place(gpu):
    # y over x or the gate, dx over dy or x: through the C entry points, as the binding allocates its own.
    x, w, b, gate = problem(50, 7, 33, torch.float16, seed=50)
    dim = 231
    y, mean, rstd = group_norm(x, w, b, gate, groups=7)
    st = torch.cuda.current_stream().cuda_stream
    for place in range(2):
        a, c = x.clone(), gate.clone()
        args = packed(abi.GROUP_NORM_STRUCT.pack, 50, dim, 7, IO_DTYPES[x.dtype], 0, 1, 1e-5, ptr(a), ptr(w), ptr(b), ptr(c),
                      ptr((a, c)[place]), 0, 0, 0, 0, dim, dim, dim, 0, 0)
        run(abi.lib().helix_group_norm_encode, 0, st, args)
        assert torch.equal((a, c)[place], y)
    dy = normal(50, dim, seed=51, dtype=torch.float16)
    want, _, _, dgate = group_norm_backward(dy, x, w, mean, rstd, b, gate, groups=7)
    for place in range(2):
        a, c, dg = x.clone(), dy.clone(), torch.empty_like(x)
        args = packed(abi.GROUP_NORM_BACKWARD_STRUCT.pack, 50, dim, 7, IO_DTYPES[x.dtype], 0, 1, 0, ptr(c), ptr(a), ptr(w),
                      ptr(b), ptr(gate), ptr(mean), ptr(rstd), ptr((a, c)[place]), ptr(dg), 0, 0, 0, 0, *[dim] * 5)
        run(abi.lib().helix_group_norm_backward_encode, 0, st, args)
        assert torch.equal((a, c)[place], want) and torch.equal(dg, dgate)


def test_rows_behind_are_left(gpu):
    # Rows of outputs are wider than the groups: what lies between them stays.
    x, w, b, _ = problem(9, 3, 35, torch.bfloat16, seed=55, gated=False)
    out = torch.full((10, 120), 3.0, device="cuda", dtype=torch.bfloat16)
    args = packed(abi.GROUP_NORM_STRUCT.pack, 9, 105, 3, IO_DTYPES[x.dtype], 0, 1, 1e-5, ptr(x), ptr(w), ptr(b), 0, ptr(out),
                  0, 0, 0, 0, 105, 0, 120, 0, 0)
    run(abi.lib().helix_group_norm_encode, 0, torch.cuda.current_stream().cuda_stream, args)
    assert torch.equal(out[:9, :105], group_norm(x, w, b, groups=3)[0])
    assert (out[:, 105:] == 3).all() and (out[9] == 3).all()


def test_other_stream_and_graph(gpu):
    x, w, b, gate = problem(300, 8, 64, torch.bfloat16, seed=60)
    dy = normal(300, 512, seed=61, dtype=torch.bfloat16)

    def step(stream=None):
        y, mean, rstd = group_norm(x, w, b, gate, groups=8, stream=stream)
        q, scale = group_norm_fp8(x, w, b, gate, groups=8, stream=stream)
        return (y, mean, rstd, q.float(), scale.float(),
                *group_norm_backward(dy, x, w, mean, rstd, b, gate, groups=8, stream=stream))

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
        x.copy_(normal(300, 512, seed=70 + k))
        graph.replay()
        torch.cuda.synchronize()
        again = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(again, step()))


def test_refusals(gpu):
    x, w = normal(4, 96), torch.ones(96, device="cuda")
    for bad in (dict(x=x.double()), dict(x=x.cpu()), dict(weight=w[:63]), dict(weight=w.half()), dict(bias=w.half()),
                dict(bias=w[1:]), dict(gate=x[:3]), dict(gate=x.half()), dict(x=normal(96, 4).t()), dict(groups=5),
                dict(groups=0), dict(groups=3.0), dict(activation="tanh"), dict(eps=1e39)):
        with pytest.raises(ValueError):
            group_norm(**{"x": x, "weight": w, "groups": 3, **bad})
    for eps in (-1.0, float("nan")):
        with pytest.raises(HelixError):
            group_norm(x, w, groups=3, eps=eps)
    wide = torch.ones(1, 19200, device="cuda")
    with pytest.raises(HelixError):
        group_norm(wide, wide[0], groups=1)
    with pytest.raises(HelixError):
        group_norm_fp8(wide, wide[0], groups=200)
    _, mean, rstd = group_norm(x, w, groups=3)
    for bad in (dict(dy=x.half()), dict(rstd=rstd[:3]), dict(mean=mean.half()), dict(mean=mean[:, :2]), dict(groups=4),
                dict(gate=x[:, :60]), dict(weight=w[1:])):
        with pytest.raises(ValueError):
            group_norm_backward(**{"dy": x, "x": x, "weight": w, "mean": mean, "rstd": rstd, "groups": 3, **bad})
