"""helix_amd.delta on the GPU against the 64-bit forms of delta_oracle.py."""
import pytest
import torch

import delta_oracle as do_
import layer_oracle as lo
from helix_amd import abi
from helix_amd.abi import HelixError
from helix_amd.delta import delta_rule, delta_rule_backward
from helix_amd.layer import IO_DTYPES, packed, ptr, run, scratch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF, NAN = float("inf"), float("nan")
NAMES = ("dq", "dk", "dv", "dg", "dbeta", "ds0")


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def problem(S, L, Hk, H, N, P, dtype, seed=0, packed_rows=False, carry=True):
    """(q, k, v, g, beta, s0): keys and queries of length one, decays from a few tokens to thousands."""
    q, k = (torch.nn.functional.normalize(normal(S, L, Hk, N, seed=seed + i), dim=-1).to(dtype) for i in range(2))
    v = normal(S, L, H, P, seed=seed + 2, dtype=dtype)
    if packed_rows:
        row = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2), v.flatten(2)[..., :3]], -1)
        q, k = row[..., :Hk * N].unflatten(-1, (Hk, N)), row[..., Hk * N:2 * Hk * N].unflatten(-1, (Hk, N))
        v = row[..., 2 * Hk * N:2 * Hk * N + H * P].unflatten(-1, (H, P))
    g = -torch.exp(1.5 * normal(H, seed=seed + 3) - 2.5) * torch.nn.functional.softplus(normal(S, L, H, seed=seed + 4))
    beta = torch.sigmoid(normal(S, L, H, seed=seed + 5))
    return q, k, v, g, beta, 0.3 * normal(S, H, N, P, seed=seed + 6) if carry else None


def check(q, k, v, g, beta, s0, scale=None, amp=None):
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    o64, states, _ = do_.forward(q, k, v, g, beta, s0, sc)
    so, ss = do_.forward_sizes(q, states, abs(sc), v.shape[2])
    o, s = delta_rule(q, k, v, g, beta, s0, scale=scale)
    assert o.dtype == v.dtype and s.dtype == torch.float32
    amp = do_.amplification(k, g, beta, v.shape[2]) if amp else 1.0
    do_.close(o, o64, so, v.dtype, "o", amp)
    do_.close(s, states[-1], ss, torch.float32, "s", amp)
    o2, s2 = delta_rule(q, k, v, g, beta, s0, scale=scale)
    assert torch.equal(o, o2) and torch.equal(s, s2)
    return o, s


def check_backward(q, k, v, g, beta, s0, ds=True, scale=None, seed=90, amp=None):
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    d = normal(*v.shape, seed=seed, dtype=v.dtype)
    S, L, H, P = v.shape
    ds = normal(S, H, q.shape[-1], P, seed=seed + 1) if ds else None
    want, size = do_.backward(d, q, k, v, g, beta, s0, ds, sc)
    got = delta_rule_backward(d, q, k, v, g, beta, s0, ds, scale=scale)
    amp = do_.amplification(k, g, beta, H) if amp else 1.0
    for n, a, b in zip(NAMES, got, want):
        assert a.dtype == (v.dtype if n in ("dq", "dk", "dv") else torch.float32)
        do_.close(a, b, size[n], a.dtype, n, amp)
    assert all(torch.equal(a, b) for a, b in zip(got, delta_rule_backward(d, q, k, v, g, beta, s0, ds, scale=scale)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [1, 2, 3, 6, 7, 12, 13, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 200, 333])
def test_lengths(gpu, L, dtype):
    p = problem(2, L, 1, 2, 64, 32, dtype, seed=L, packed_rows=L % 2 == 1, carry=L % 3 != 0)
    check(*p)
    check_backward(*p, ds=L % 4 != 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,P", [(1, 1), (2, 3), (5, 7), (8, 64), (31, 17), (40, 72), (63, 15), (64, 128), (65, 16), (66, 33),
                                 (100, 130), (127, 65), (128, 192), (128, 1)])
@pytest.mark.parametrize("L", [5, 9, 100])
def test_widths(gpu, L, N, P, dtype):
    p = problem(1, L, 2, 2, N, P, dtype, seed=N + P, packed_rows=(N + P) % 2 == 0)
    check(*p)
    check_backward(*p)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,Hk,H", [(1, 1, 1), (3, 1, 5), (2, 3, 3), (1, 4, 12), (5, 2, 16)])
@pytest.mark.parametrize("L", [1, 90])
def test_heads(gpu, S, Hk, H, L, dtype):
    p = problem(S, L, Hk, H, 48, 24, dtype, seed=H)
    check(*p)
    check_backward(*p)


@pytest.mark.parametrize("S,L,Hk,H,N,P,dtype", [(1, 1500, 2, 4, 128, 64, torch.bfloat16), (3, 1003, 2, 2, 64, 48, torch.float32),
                                                (1, 2050, 1, 1, 96, 20, torch.float16), (64, 1, 2, 8, 128, 64, torch.bfloat16),
                                                (1, 70, 1, 1, 128, 65536, torch.bfloat16), (1, 2, 1, 2, 128, 65535, torch.float16),
                                                (1, 66, 1, 8192, 1, 1, torch.float32), (70000, 7, 1, 1, 2, 2, torch.bfloat16)])
def test_long_and_many(gpu, S, L, Hk, H, N, P, dtype):
    p = problem(S, L, Hk, H, N, P, dtype, seed=7)
    check(*p)
    check_backward(*p)


# Long calls of some heads go in segments whose operands are formed while the one before is walked.
@pytest.mark.parametrize("S,L,Hk,H,N,P,dtype", [(1, 6200, 2, 64, 8, 8, torch.bfloat16), (1, 6145, 64, 64, 66, 17, torch.float16),
                                                (2, 6300, 3, 48, 16, 24, torch.bfloat16), (1, 12800, 16, 32, 65, 4, torch.bfloat16)])
def test_segments_ahead(gpu, S, L, Hk, H, N, P, dtype):
    check(*problem(S, L, Hk, H, N, P, dtype, seed=L, packed_rows=S == 1))


def test_segments_ahead_in_place_and_captured(gpu):
    # The state goes from segment to segment through s, which may be s0; a graph's segments follow each other on every replay.
    q, k, v, g, beta, s0 = problem(1, 6211, 2, 64, 24, 16, torch.bfloat16, seed=80)
    o, s = delta_rule(q, k, v, g, beta, s0)
    state, out = s0.clone(), torch.empty_like(o)
    encode(q, k, v, g, beta, state, out, state)
    assert torch.equal(out, o) and torch.equal(state, s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = delta_rule(q, k, v, g, beta, s0)
    for i in range(3):
        v.copy_(normal(*v.shape, seed=81 + i, dtype=v.dtype))
        eager = [t.clone() for t in delta_rule(q, k, v, g, beta, s0)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


@pytest.mark.parametrize("L,tok,seq", [(300, (1 << 23) + 24, 64), (3, 200, (1 << 31) + 72), (70, 200, (1 << 31) + 72)])
def test_offsets_past_32_bits(gpu, L, tok, seq):
    # Tokens, or sequences, that lie gigabytes apart in one buffer; only what belongs to them is written.
    S, Hk, H, N, P = 2, 1, 2, 24, 32
    p = problem(S, L, Hk, H, N, P, torch.bfloat16, seed=95)
    d = normal(S, L, H, P, seed=96, dtype=torch.bfloat16)
    want, grads = delta_rule(*p), delta_rule_backward(d, *p)
    q, k, v, g, beta, s0 = p
    if seq < tok:
        seq *= 3   # (the sequences' rows side by side)
    buf = torch.empty((S - 1) * seq + L * tok, dtype=torch.bfloat16, device="cuda")

    def place(t, at):
        heads, width = t.shape[2:]
        view = buf.as_strided((S, L, heads, width), (seq, tok, width, 1), at)
        view.copy_(t)
        return view

    far = [place(t, at) for t, at in ((q, 0), (k, N), (v, 2 * N))]
    got = delta_rule(*far, g, beta, s0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(delta_rule_backward(d, *far, g, beta, s0), grads))
    out = buf.as_strided((S, L, H, P), (seq, tok, P, 1), 2 * N)   # (over v's place, which another copy of it then is read from)
    state = torch.empty_like(want[1])
    encode(far[0], far[1], v, g, beta, s0, out, state)
    assert torch.equal(out, want[0]) and torch.equal(state, want[1]) and torch.equal(far[0], q) and torch.equal(far[1], k)


# Where many heads share the machine, more tokens go one by one: up to 32 in fp32, more than LDS has the keys of at a time.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,L,Hk,H,N,P", [(4, 10, 4, 64, 32, 16), (4, 11, 4, 64, 32, 16), (4, 20, 4, 64, 32, 16), (4, 21, 4, 64, 32, 16),
                                          (6, 16, 8, 64, 24, 20), (6, 17, 8, 64, 24, 20), (3, 32, 8, 64, 40, 72), (6, 33, 8, 64, 24, 20)])
def test_some_tokens_of_many_heads(gpu, S, L, Hk, H, N, P, dtype):
    check(*problem(S, L, Hk, H, N, P, dtype, seed=L, packed_rows=L % 2 == 0))


def test_scale(gpu):
    p = problem(1, 80, 1, 2, 32, 16, torch.float32, seed=3)
    for scale in (1.0, -0.7, 0.0):
        check(*p, scale=scale)
        check_backward(*p, scale=scale)


@pytest.mark.parametrize("L", [5, 10, 150])
def test_long_memory(gpu, L):
    # No decay at all, and a state that is large against what the tokens bring.
    q, k, v, g, beta, s0 = problem(1, L, 2, 2, 64, 32, torch.bfloat16, seed=8)
    check(q, k, v, torch.zeros_like(g), beta, 100 * s0)
    check_backward(q, k, v, torch.zeros_like(g), beta, 100 * s0)


@pytest.mark.parametrize("L", [8, 190])
@pytest.mark.parametrize("beta_is", [0.0, 1.0, 2.0])
def test_keys_that_repeat(gpu, L, beta_is):
    # The same key again and again: the entries of A are as large as they get, and beta = 2 reflects.
    q, k, v, g, beta, s0 = problem(1, L, 1, 2, 32, 16, torch.float32, seed=9)
    k = k[:, :1].expand(1, L, 1, 32)
    g = 0.01 * g
    check(q, k, v, g, torch.full_like(beta, beta_is), s0, amp=True)
    check_backward(q, k, v, g, torch.full_like(beta, beta_is), s0, amp=True)


@pytest.mark.parametrize("L", [12, 200])
def test_decays_at_the_ends(gpu, L):
    # -inf and the type's lowest value forget all before; strong decays leave nothing of a chunk's start; 0 keeps.
    q, k, v, g, beta, s0 = problem(2, L, 1, 3, 40, 20, torch.float32, seed=10)
    lowest = torch.finfo(torch.float32).min
    g[0, 5, 0], g[0, L // 2, 0], g[1, L - 2, 1], g[0, 0, 2], g[1, L // 2:L // 2 + 3, 2] = -INF, lowest, -INF, lowest, -INF
    g[1, :, 0] = -30.0
    g[1, 3:6, 1] = 0.0
    check(q, k, v, g, beta, s0)
    check_backward(q, k, v, g, beta, s0)
    o, s = delta_rule(q, k, v, g, beta, s0)
    assert o.isfinite().all() and s.isfinite().all()
    # What came before a token that forgets does not reach what follows.
    cut = L // 2
    o2, s2 = delta_rule(q[:1, cut:], k[:1, cut:], v[:1, cut:], g[:1, cut:], beta[:1, cut:], None)
    assert (o[0, cut:, 0] - o2[0, :, 0]).abs().max() < 1e-5 and (s[0, 0] - s2[0, 0]).abs().max() < 1e-5


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_that_leave_the_state(gpu, dtype):
    # Sequences of different lengths in one batch: g = 0 and beta = 0 behind their ends.
    q, k, v, g, beta, s0 = problem(3, 150, 2, 2, 64, 32, dtype, seed=11)
    ends = (150, 70, 0)
    for i, n in enumerate(ends):
        g[i, n:], beta[i, n:] = 0.0, 0.0
    o, s = check(q, k, v, g, beta, s0)
    assert torch.equal(s[2], s0[2])
    o1, s1 = delta_rule(q[1:2, :70], k[1:2, :70], v[1:2, :70], g[1:2, :70], beta[1:2, :70], s0[1:2])
    assert torch.equal(o1, o[1:2, :70]) and torch.equal(s1, s[1:2])


def test_steps_and_chunks_agree(gpu):
    # One by one, in pieces and all at once: the state that one call leaves is the next one's.
    q, k, v, g, beta, s0 = problem(2, 200, 2, 4, 128, 64, torch.float32, seed=12)
    o, s = delta_rule(q, k, v, g, beta, s0)
    for cuts in ([1] * 40, [7, 16, 17, 64, 96], [100, 100]):
        at, state, outs = 0, s0, []
        for n in cuts:
            part, state = delta_rule(*(t[:, at:at + n] for t in (q, k, v, g, beta)), state)
            outs.append(part)
            at += n
        assert (torch.cat(outs, 1) - o[:, :at]).norm() <= 1e-6 * o[:, :at].norm()
        if at == 200:
            assert (state - s).norm() <= 1e-6 * s.norm()


@pytest.mark.parametrize("L", [5, 170])
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
def test_what_is_not_finite_stays_in_its_head(gpu, L, bad):
    p = problem(2, L, 2, 4, 64, 48, torch.bfloat16, seed=13)
    d = normal(2, L, 4, 48, seed=14, dtype=torch.bfloat16)
    o, s = delta_rule(*p)
    grads = delta_rule_backward(d, *p)
    at = L - 2
    first = at // 64 * 64 if L > 16 else at
    # An element of v: its column, from its chunk on.
    q, k, v, g, beta, s0 = p
    v2 = v.clone()
    v2[1, at, 2, 5] = bad
    o2, s2 = delta_rule(q, k, v2, g, beta, s0)
    assert not o2[1, at:, 2, 5].isfinite().any() and not s2[1, 2, :, 5].isfinite().all()
    keep = torch.ones_like(o2, dtype=torch.bool)
    keep[1, first:, 2, 5] = False
    assert torch.equal(o2[keep], o[keep])
    s2[1, 2, :, 5] = s[1, 2, :, 5]
    assert torch.equal(s2, s)
    # A key: the value heads that share it.
    k2 = k.clone()
    k2[0, at, 1, 3] = bad
    o2, s2 = delta_rule(q, k2, v, g, beta, s0)
    assert not o2[0, at:, 2:].isfinite().any() and not s2[0, 2:].isfinite().all()
    assert torch.equal(o2[1], o[1]) and torch.equal(o2[0, :, :2], o[0, :, :2]) and torch.equal(o2[0, :first], o[0, :first])
    assert torch.equal(s2[1], s[1]) and torch.equal(s2[0, :2], s[0, :2])
    got = delta_rule_backward(d, q, k2, v, g, beta, s0)
    for n, a, b in zip(NAMES, got, grads):
        assert torch.equal(a[1], b[1]), n
        if n in ("dq", "dk"):
            assert torch.equal(a[0, :, 0], b[0, :, 0]), n
        elif n == "ds0":
            assert torch.equal(a[0, :2], b[0, :2]), n
        else:
            assert torch.equal(a[0, :, :2], b[0, :, :2]), n


def test_strides(gpu):
    # Heads outside tokens, sequences inside, one row for all tokens; unaligned starts.
    S, L, H, N, P = 2, 70, 3, 24, 40
    base = normal(H, L, S, N + 5, seed=20, dtype=torch.bfloat16) / 5
    q, k = base[..., 1:N + 1].permute(2, 1, 0, 3), base[..., 5:N + 5].permute(2, 1, 0, 3)
    v = normal(S, 1, H, P + 1, seed=21, dtype=torch.bfloat16)[..., 1:].expand(S, L, H, P)
    gb = -torch.rand(S, L, 2 * H + 1, device="cuda")
    g, beta = gb[..., 1:H + 1], -gb[..., H + 1:]
    for n in (9, L):
        check(*(t[:, :n] for t in (q, k, v, g, beta)), None)
        check_backward(*(t[:, :n] for t in (q, k, v, g, beta)), None)


def encode(q, k, v, g, beta, s0, o, s, nbytes=None):
    S, L, Hk, N = q.shape
    H, P = v.shape[2:]
    st = torch.cuda.current_stream().cuda_stream

    def pack(buf, n):
        return packed(abi.DELTA_RULE_STRUCT.pack, S, L, Hk, H, N, P, IO_DTYPES[q.dtype], N ** -0.5, ptr(q), ptr(k), ptr(v), ptr(g),
                      ptr(beta), ptr(s0), ptr(o), ptr(s), buf, n, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
                      *g.stride()[:2], *beta.stride()[:2], *o.stride()[:3])

    lib = abi.lib()
    need = lib.helix_delta_rule_scratch_size(pack(0, 0))
    run(lib.helix_delta_rule_encode, 0, st, pack(ptr(scratch(0, st, None, need)), need))


@pytest.mark.parametrize("L", [0, 1, 16, 100, 130])
def test_state_in_place(gpu, L):
    # s over s0, ds0 over d_s; outputs with heads outside tokens, and what lies between them stays.
    q, k, v, g, beta, s0 = problem(2, L, 1, 2, 40, 24, torch.bfloat16, seed=22)
    o, s = delta_rule(q, k, v, g, beta, s0)
    state = s0.clone()
    out = torch.full((2, 2, L + 1, 30), 3.0, device="cuda", dtype=torch.bfloat16)
    encode(q, k, v, g, beta, state, out[:, :, :L, 2:26].transpose(1, 2), state)
    assert torch.equal(state, s) and torch.equal(out[:, :, :L, 2:26].transpose(1, 2), o)
    assert (out[:, :, L] == 3).all() and (out[..., :2] == 3).all() and (out[..., 26:] == 3).all()
    d, ds = normal(2, L, 2, 24, seed=23, dtype=torch.bfloat16), normal(2, 2, 40, 24, seed=24)
    want = delta_rule_backward(d, q, k, v, g, beta, s0, ds)
    if L == 0:
        assert torch.equal(s, s0) and torch.equal(want[5], ds)
    got = [torch.empty_like(t) for t in want[:5]]
    place = ds.clone()
    lib, st = abi.lib(), torch.cuda.current_stream().cuda_stream

    def pack(buf, n):
        return abi.DELTA_RULE_BACKWARD_STRUCT.pack(2, L, 1, 2, 40, 24, 2 if q.dtype == torch.bfloat16 else 0, 40 ** -0.5, ptr(d),
                                                   ptr(q), ptr(k), ptr(v), ptr(g), ptr(beta), ptr(s0), ptr(place),
                                                   *[ptr(t) for t in got], ptr(place), buf, n, *d.stride()[:3], *q.stride()[:3],
                                                   *k.stride()[:3], *v.stride()[:3], *g.stride()[:2], *beta.stride()[:2])

    need = lib.helix_delta_rule_backward_scratch_size(pack(0, 0))
    run(lib.helix_delta_rule_backward_encode, 0, st, pack(ptr(scratch(0, st, None, need)), need))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(place, want[5])


def test_segments(gpu):
    # Calls whose operands pass the scratch limit go in segments: 3000 sequences of a few chunks, against some of them alone.
    S, L, H, N, P = 3000, 200, 8, 16, 16
    p = problem(S, L, 1, H, N, P, torch.bfloat16, seed=25)
    d, ds = normal(S, L, H, P, seed=26, dtype=torch.bfloat16), normal(S, H, N, P, seed=27)
    o, s = delta_rule(*p)
    grads = delta_rule_backward(d, *p, ds)
    for i in (0, 1234, S - 1):
        one = [t[i:i + 1] for t in p]
        o1, s1 = delta_rule(*one)
        assert torch.equal(o1, o[i:i + 1]) and torch.equal(s1, s[i:i + 1])
        for n, a, b in zip(NAMES, delta_rule_backward(d[i:i + 1], *one, ds[i:i + 1]), grads):
            assert torch.equal(a, b[i:i + 1]), n


def test_against_differences(gpu):
    # Central differences of the 64-bit forward in random directions.
    p = problem(1, 70, 1, 2, 12, 10, torch.float32, seed=30)
    do, ds = normal(1, 70, 2, 10, seed=31), normal(1, 2, 12, 10, seed=32)
    got = delta_rule_backward(do, *p, ds)
    at = [lo.f64(t) for t in p]

    def loss(*x):
        o, states, _ = do_.forward(*x, 12 ** -0.5)
        return float((lo.f64(do) * o).sum() + (lo.f64(ds) * states[-1]).sum())

    for seed in range(4):
        way = [lo.f64(normal(*t.shape, seed=40 + 6 * seed + i)) for i, t in enumerate(at)]
        e = 1e-5
        num = (loss(*[t + e * w for t, w in zip(at, way)]) - loss(*[t - e * w for t, w in zip(at, way)])) / (2 * e)
        ana = sum(float((lo.f64(a) * w).sum()) for a, w in zip(got, way))
        size = sum(float((lo.f64(a) * w).abs().sum()) for a, w in zip(got, way))
        assert abs(num - ana) <= 1e-5 * size


def test_empty(gpu):
    for S, H in ((0, 2), (2, 0)):
        q = torch.empty(S, 5, min(H, 1), 8, device="cuda")
        v, g = torch.empty(S, 5, H, 4, device="cuda"), torch.empty(S, 5, H, device="cuda")
        o, s = delta_rule(q, q, v, g, g)
        assert o.shape == (S, 5, H, 4) and s.shape == (S, H, 8, 4)
        assert [t.shape for t in delta_rule_backward(v, q, q, v, g, g)] == [q.shape, q.shape, v.shape, g.shape, g.shape, s.shape]


def test_other_stream_and_graph(gpu):
    for L in (1, 100):
        q, k, v, g, beta, s0 = problem(2, L, 2, 4, 64, 32, torch.bfloat16, seed=50)
        d, ds = normal(2, L, 4, 32, seed=51, dtype=torch.bfloat16), normal(2, 4, 64, 32, seed=52)

        def step(stream=None):
            return (*delta_rule(q, k, v, g, beta, s0, stream=stream),
                    *delta_rule_backward(d, q, k, v, g, beta, s0, ds, stream=stream))

        want = step()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = step(side)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        # Two graphs, replayed in turn with eager calls between: neither shares scratch with the other.
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
            graphs.append((graph, out))
        for i in range(3):
            v.copy_(normal(2, L, 4, 32, seed=60 + i))
            eager = [t.clone() for t in step()]
            for graph, out in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for _, out in graphs:
                assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_two_streams_at_once(gpu):
    a, b = problem(1, 300, 2, 4, 128, 64, torch.bfloat16, seed=70), problem(1, 300, 2, 4, 128, 64, torch.bfloat16, seed=71)
    d = normal(1, 300, 4, 64, seed=72, dtype=torch.bfloat16)
    want = [(*delta_rule(*p), *delta_rule_backward(d, *p)) for p in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i, p in enumerate((a, b)):
            got[i] = (*delta_rule(*p, stream=streams[i]), *delta_rule_backward(d, *p, stream=streams[i]))
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert all(torch.equal(s, t) for s, t in zip(x, y))


def test_refusals(gpu):
    q, k, v, g, beta, s0 = problem(2, 20, 2, 4, 16, 8, torch.float32, seed=80)
    good = dict(q=q, k=k, v=v, g=g, beta=beta, s0=s0)
    for bad in (dict(q=q.double()), dict(q=q.cpu()), dict(q=q[0]), dict(v=v[0]), dict(k=k.half()), dict(k=k[:, :19]),
                dict(v=v.half()), dict(v=v[:, :, :3]), dict(g=g.half()), dict(g=g[:, :, :2]), dict(beta=beta[:1]),
                dict(beta=beta.double()), dict(s0=s0.half()), dict(s0=s0[:1]), dict(s0=s0.transpose(2, 3).contiguous().transpose(2, 3)),
                dict(q=q.transpose(2, 3).contiguous().transpose(2, 3)), dict(q=q[:, :, :0], k=k[:, :, :0]),
                dict(g=g.transpose(1, 2).contiguous().transpose(1, 2)), dict(q=q[..., :0], k=k[..., :0]), dict(scale=1e39)):
        with pytest.raises(ValueError):
            delta_rule(**{**good, **bad})
        with pytest.raises(ValueError):
            delta_rule_backward(v, **{**good, **bad})
    for bad in (dict(do=v[:, :3]), dict(do=v.half()), dict(ds=s0.half()), dict(ds=s0[:, :1])):
        with pytest.raises(ValueError):
            delta_rule_backward(**{"do": v, **good, **bad})
    wide = torch.ones(1, 2, 1, 129, device="cuda")
    with pytest.raises(HelixError):
        delta_rule(wide, wide, wide, torch.zeros(1, 2, 1, device="cuda"), torch.zeros(1, 2, 1, device="cuda"))
    with pytest.raises(HelixError):
        delta_rule(q, k, v, g, beta, scale=NAN)
