"""helix_amd.recurrence on the GPU against the 64-bit forms of layer_oracle.py."""
import pytest
import torch

import layer_oracle as lo
from helix_amd.recurrence import gated_scan, gated_scan_backward

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = float("inf")


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def problem(S, L, D, dtype=torch.float32, seed=0, packed=False, carry=True, mean=2.0):
    if packed:
        row = normal(S, L, 2 * D + 8, seed=seed, dtype=dtype)
        g, v = row[..., :D], row[..., D:2 * D]
        g.mul_(1.5).add_(mean)
    else:
        g, v = (mean + 1.5 * normal(S, L, D, seed=seed)).to(dtype), normal(S, L, D, seed=seed + 1, dtype=dtype)
    return g, v, normal(S, D, seed=seed + 2) if carry else None


def check(g, v, h0, seed=90):
    h64, last64 = lo.scan(g, v, h0)
    bh, bl = lo.scan_bound(g, v, h0, h64)
    h, last = gated_scan(g, v, h0)
    lo.within(h, h64, bh, "h")
    lo.within(last, last64, bl, "last")
    dh, dl = normal(*g.shape, seed=seed, dtype=g.dtype), normal(g.shape[0], g.shape[2], seed=seed + 1)
    dl = dl if h0 is not None else None
    want = lo.scan_backward(dh, g, v, h, h0, dl)
    bounds = lo.scan_backward_bound(dh, g, v, h, h0, dl, want[0], want[1])
    got = gated_scan_backward(dh, g, v, h, h0, dl)
    for name, a, b, c in zip(("dg", "dv", "dh0"), got, want, bounds):
        lo.within(a, b, c, name)
    # The same again: no order of arrival enters.
    assert torch.equal(h, gated_scan(g, v, h0)[0])
    assert all(torch.equal(a, b) for a, b in zip(got, gated_scan_backward(dh, g, v, h, h0, dl)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [1, 2, 3, 7, 16, 31, 64, 65, 127, 200, 513, 1000])
def test_lengths(gpu, L, dtype):
    check(*problem(2, L, 136, dtype, seed=L, packed=L % 2 == 0, carry=L % 3 != 0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 3, 8, 33, 63, 64, 65, 127, 128, 130, 256, 520])
def test_channels(gpu, D, dtype):
    check(*problem(3, 150, D, dtype, seed=D, packed=D % 2 == 1))


@pytest.mark.parametrize("S,L,D,dtype", [(1, 8192, 64, torch.bfloat16), (1, 20011, 40, torch.float32),
                                         (2, 4096, 200, torch.bfloat16), (1, 5000, 1001, torch.float16),
                                         (300, 9, 72, torch.bfloat16), (64, 1, 4096, torch.bfloat16),
                                         (5, 2049, 96, torch.float32)])
def test_long_and_many(gpu, S, L, D, dtype):
    check(*problem(S, L, D, dtype, seed=7, packed=True))


@pytest.mark.parametrize("L", [40, 700, 3000])
def test_long_memory(gpu, L):
    # Gates near 1: the state of the first token reaches the last one.
    g, v, h0 = problem(1, L, 100, seed=8, mean=12.0)
    check(g, v, 100 * h0)
    check(*problem(1, L, 100, seed=9, mean=-12.0))


def test_gates_at_the_ends(gpu):
    g, v, h0 = problem(2, 600, 70, seed=10)
    g[0, 100:500] = INF      # keeps the state over whole parts of the sequence
    g[1, 250] = -INF         # takes v alone
    g[:, :, 5] = INF         # a channel that takes one token alone
    g[:, :, 6] = -INF
    g[:, 30] = 3e38
    g[:, 31] = -3e38
    check(g, v, h0)
    h, last = gated_scan(g, v, h0)
    # Channel 5: what came in up to token 31, which takes v alone, and that from there on.
    assert torch.equal(h[:, :31, 5], h0[:, None, 5].expand(2, 31))
    assert torch.equal(h[:, 31:, 5], v[:, 31:32, 5].expand(2, 569)) and torch.equal(last[:, 5], v[:, 31, 5])


def test_nan_stays_in_its_channel(gpu):
    for spot in ("g", "v"):
        g, v, h0 = problem(2, 900, 80, seed=11)
        want, _ = gated_scan(g, v, h0)
        (g if spot == "g" else v)[1, 400, 33] = float("nan")
        got, last = gated_scan(g, v, h0)
        assert torch.isnan(got[1, 400:, 33]).all() and torch.isnan(last[1, 33])
        got[1, 400:, 33] = want[1, 400:, 33]
        assert torch.equal(got, want)
        dh = normal(2, 900, 80, seed=12)
        dg, dv, dh0 = gated_scan_backward(dh, g, v, got, h0)
        clean = [t.clone() for t in (dg, dv)]
        assert all(torch.isfinite(t[:, :, torch.arange(80) != 33]).all() for t in clean) and torch.isnan(dg[1, 400, 33])
        assert torch.isfinite(dh0[0]).all()


def test_strides(gpu):
    # Token-major storage, broadcast gates, reversed roles of sequence and token strides, odd offsets.
    base = normal(300, 3, 70, seed=13)
    check(base.transpose(0, 1), normal(3, 300, 70, seed=14), None)
    check(normal(1, 1, 70, seed=15).expand(2, 257, 70), normal(2, 257, 70, seed=16), normal(2, 70, seed=17))
    wide = normal(2, 260, 211, seed=18, dtype=torch.bfloat16)
    check(wide[:, :, 3:100], wide[:, :, 101:198], normal(2, 97, seed=19))
    check(wide[:, :, 3:99], wide[:, :, 102:198], normal(2, 96, seed=19))
    check(wide[:, :9, 1:129], wide[:, :9, 2:130], normal(2, 128, seed=19))


def test_rows_far_apart(gpu):
    # Sequences more than 2^32 bytes apart, and tokens so far apart that a wave's reach past 2^29 bytes.
    far = torch.empty(2, (1 << 31) + 64, device="cuda", dtype=torch.bfloat16)
    g, v = (far[:, k * 4096:k * 4096 + 40 * 64].unflatten(1, (40, 64)) for k in (0, 1))
    g.copy_(2 + normal(2, 40, 64, seed=70))
    v.copy_(normal(2, 40, 64, seed=71))
    check(g, v, normal(2, 64, seed=72))
    del far, g, v
    far = torch.empty(20, 9_000_000, device="cuda", dtype=torch.bfloat16)
    g, v = (far[None, :, k * 4096:k * 4096 + 72] for k in (0, 1))
    g.copy_(2 + normal(1, 20, 72, seed=73))
    v.copy_(normal(1, 20, 72, seed=74))
    check(g, v, normal(1, 72, seed=75))


def test_parts_join_as_one(gpu):
    # A sequence in two calls, the state carried: the same values as in one, up to the roundings of the joins.
    g, v, h0 = problem(2, 1200, 64, seed=20)
    h, last = gated_scan(g, v, h0)
    h1, mid = gated_scan(g[:, :511], v[:, :511], h0)
    h2, end = gated_scan(g[:, 511:], v[:, 511:], mid)
    h64, last64 = lo.scan(g, v, h0)
    bh, bl = lo.scan_bound(g, v, h0, h64)
    lo.within(torch.cat([h1, h2], 1), h64, bh)
    lo.within(end, last64, bl)


def test_gradients_against_differences(gpu):
    S, L, D = 2, 90, 5
    g, v, h0 = problem(S, L, D, seed=21, mean=1.0)
    ch, cl = normal(S, L, D, seed=24), normal(S, D, seed=25)
    h, _ = gated_scan(g, v, h0)
    grads = [lo.f64(t) for t in gated_scan_backward(ch, g, v, h, h0, cl)]

    def loss(g, v, h0):
        h, last = lo.scan(g, v, h0)
        return float((lo.f64(ch) * h).sum() + (lo.f64(cl) * last).sum())

    for seed in range(4):
        dirs = [lo.f64(normal(*t.shape, seed=60 + 3 * seed + i)) for i, t in enumerate((g, v, h0))]
        at = [lo.f64(t) for t in (g, v, h0)]
        d = 1e-5
        num = (loss(*(a + d * p for a, p in zip(at, dirs))) - loss(*(a - d * p for a, p in zip(at, dirs)))) / (2 * d)
        ana = sum(float((a * p).sum()) for a, p in zip(grads, dirs))
        size = sum(float((a * p).abs().sum()) for a, p in zip(grads, dirs))
        assert abs(num - ana) <= 2e-6 * size    # fp32 gradients over 90 steps; d^2 of the differences


def test_empty(gpu):
    e = torch.empty(2, 0, 16, device="cuda")
    h0 = normal(2, 16, seed=30)
    h, last = gated_scan(e, e, h0)
    assert h.shape == (2, 0, 16) and torch.equal(last, h0)
    assert (gated_scan(e, e)[1] == 0).all()
    dg, dv, dh0 = gated_scan_backward(e, e, e, e, h0, h0)
    assert dg.shape == (2, 0, 16) and torch.equal(dh0, h0)
    n = torch.empty(0, 5, 16, device="cuda")
    assert gated_scan(n, n)[0].shape == (0, 5, 16)


@pytest.mark.parametrize("L", [1, 300, 3000])
def test_other_stream_and_graph(gpu, L):
    g, v, h0 = problem(2, L, 200, torch.bfloat16, seed=31)
    dh = normal(2, L, 200, seed=34, dtype=torch.bfloat16)

    def step(stream=None):
        h, last = gated_scan(g, v, h0, stream=stream)
        return (h, last, *gated_scan_backward(dh, g, v, h, h0, last, stream=stream))

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        v.copy_(normal(2, L, 200, seed=40 + k))
        graph.replay()
        torch.cuda.synchronize()
        again = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(again, step()))


def test_refusals(gpu):
    g, v, h0 = problem(2, 10, 16)
    for bad in (dict(g=g.double()), dict(v=v.half()), dict(v=v[:, :9]), dict(h0=h0.half()), dict(h0=h0[:1]),
                dict(g=g.cpu()), dict(g=g[0]), dict(h0=normal(16, 2).t()), dict(g=normal(2, 16, 10).transpose(1, 2))):
        with pytest.raises(ValueError):
            gated_scan(**{"g": g, "v": v, "h0": h0, **bad})
    h, _ = gated_scan(g, v, h0)
    for bad in (dict(dh=h.half()), dict(h=h[:, 1:]), dict(dh_last=h0[:, 1:]), dict(h0=h0.double())):
        with pytest.raises(ValueError):
            gated_scan_backward(**{"dh": h, "g": g, "v": v, "h": h, "h0": h0, **bad})
