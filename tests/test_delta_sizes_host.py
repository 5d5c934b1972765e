"""What the delta rule's scratch sizes are for every size that an argument can have, without a GPU."""
import itertools

import pytest

from helix_amd import abi
from helix_amd.desc import HELIX_ERR_NO_DEVICE, HELIX_ERR_UNSUPPORTED_SHAPE

I32 = 2 ** 31 - 1


def forward(S, L, Hk, H, N, P, io=2):
    return abi.DELTA_RULE_STRUCT.pack(S, L, Hk, H, N, P, io, 1.0, *[0] * 26)


def backward(S, L, Hk, H, N, P, io=2):
    return abi.DELTA_RULE_BACKWARD_STRUCT.pack(S, L, Hk, H, N, P, io, 1.0, *[0] * 32)


def sizes(*a):
    lib = abi.lib()
    return lib.helix_delta_rule_scratch_size(forward(*a)), lib.helix_delta_rule_backward_scratch_size(backward(*a))


# Heads of queries that do not divide those of values: a call refuses them, whatever products they would make.
@pytest.mark.parametrize("a", [(1 << 30, 100, 4194301, 1, 128, 3), (1 << 30, 100, I32, 1, 128, 3), (4, 100, 3, 4, 64, 64),
                               (4, 100, 8, 4, 64, 64), (4, 100, 0, 4, 64, 64), (4, 100, -4, 4, 64, 64)])
def test_heads_that_are_refused_need_none(a):
    assert sizes(*a) == (0, 0)


def test_every_size_has_an_answer():
    edge = (-I32 - 1, -1, 0, 1, 2, 100, 4194301, 1 << 30, I32)
    for S, L, Hk, H in itertools.product(edge, repeat=4):
        for N, P in ((1, 1), (128, 3), (128, 1 << 16), (129, 1), (I32, I32), (0, 0)):
            sizes(S, L, Hk, H, N, P)


GIB = 1 << 30


# Many sequences, heads and tokens at once, each and together.
@pytest.mark.parametrize("io", [0, 2])
@pytest.mark.parametrize("a", [(64, 4096, 8, 64, 128, 64), (64, 8192, 4, 32, 128, 128), (256, 4096, 4, 32, 128, 128), (64, 8192, 8, 64, 128, 64),
                               (64, 2048, 8, 64, 128, 64), (32, 4096, 8, 64, 128, 128), (256, 2048, 8, 64, 128, 128), (8, 1 << 17, 16, 64, 128, 64),
                               (1, 1 << 20, 128, 128, 128, 128), (1, 1 << 21, 8, 64, 128, 64), (2, 1 << 22, 4, 4, 128, 256), (1, 4096, 2, 2, 128, 1 << 14),
                               (100000, 100, 1, 2, 16, 16), (2, 200, 1000, 8000, 40, 24), (1 << 20, 65, 1, 1, 128, 64), (3, 16000, 100, 300, 16, 16)])
def test_backward_scratch_stays_bounded(a, io):
    assert 0 < sizes(*a, io)[1] <= 3 * GIB


@pytest.mark.parametrize("io", [0, 2])
@pytest.mark.parametrize("a", [(3000, 200, 1, 16, 16, 16), (100000, 100, 1, 2, 16, 16), (1, 70, 1, 40000, 128, 64), (1, 1 << 20, 40000, 40000, 16, 16),
                               (1 << 20, 65, 64, 64, 128, 64), (1, 1 << 21, 8, 64, 128, 64), ((1 << 31) - 1, 100, 1, 1, 1, 1)])
def test_forward_scratch_stays_bounded(a, io):
    assert 0 < sizes(*a, io)[0] <= GIB


# A launch holds 2^32 threads; calls of more heads than that go in parts. Only heads that share one of the queries' stay
# together, backward.
@pytest.mark.parametrize("a,status", [((1 << 25, 3, 1, 1, 8, 8), (HELIX_ERR_NO_DEVICE,) * 2), ((1 << 25, 70, 1, 1, 8, 8), (HELIX_ERR_NO_DEVICE,) * 2),
                                      ((1, 1, 1 << 25, 1 << 25, 8, 8), (HELIX_ERR_NO_DEVICE, HELIX_ERR_UNSUPPORTED_SHAPE)),   # (dv's rows: 2^31 bytes)
                                      ((1, 1, 1, (1 << 23) - 1, 8, 1), (HELIX_ERR_NO_DEVICE, HELIX_ERR_UNSUPPORTED_SHAPE)),
                                      ((1, 1, 1, 6710886, 8, 1), (HELIX_ERR_NO_DEVICE,) * 2), ((1, 0, 1, 6710886, 8, 1), (HELIX_ERR_NO_DEVICE,) * 2),
                                      ((1, 0, 1, 6710887, 8, 1), (HELIX_ERR_NO_DEVICE, HELIX_ERR_UNSUPPORTED_SHAPE)),
                                      ((1, 1, 1, 6710887, 8, 1), (HELIX_ERR_NO_DEVICE, HELIX_ERR_UNSUPPORTED_SHAPE)),
                                      ((300, 70, 16, 64, 128, 1 << 16), (HELIX_ERR_NO_DEVICE,) * 2)])
def test_heads_of_more_than_one_launch(a, status):
    S, L, Hk, H, N, P = a
    host, lib = abi.Context(host_only=True), abi.lib()
    at = 1 << 12   # an address that nothing reads
    qk, v, g = (L * Hk * N, Hk * N, N), (L * H * P, H * P, P), (L * H, H)
    strides = (*qk, *qk, *v, *g, *g)
    fwd = abi.DELTA_RULE_STRUCT.pack(*a, 2, 1.0, *[at] * 5, 0, *[at] * 3, 1 << 50, *strides, *v)
    bwd = abi.DELTA_RULE_BACKWARD_STRUCT.pack(*a, 2, 1.0, *[at] * 15, 1 << 50, *v, *strides)
    got = tuple(int(f(host.handle, None, x)) for f, x in ((lib.helix_delta_rule_encode, fwd), (lib.helix_delta_rule_backward_encode, bwd)))
    host.close()
    assert got == status


def test_gates_at_any_distance():
    # What 64 tokens of q, k, v and o span is bounded, of g and beta it is not: 2^23 heads and more of two tokens are taken.
    host, lib = abi.Context(host_only=True), abi.lib()
    at, H = 1 << 12, 1 << 23
    far = 1 << 40
    for a, gate in (((1, 2, 1, H, 8, 1), (2 * H, H)), ((2, 100, 2, 4, 16, 8), (far, far // 200)), ((2, 5, 2, 4, 16, 8), (4, far))):
        S, L, Hk, H_, N, P = a
        qk, v = (L * Hk * N, Hk * N, N), (L * H_ * P, H_ * P, P)
        strides = (*qk, *qk, *v, *gate, *gate)
        fwd = abi.DELTA_RULE_STRUCT.pack(*a, 2, 1.0, *[at] * 5, 0, *[at] * 3, 1 << 50, *strides, *v)
        assert int(lib.helix_delta_rule_encode(host.handle, None, fwd)) == HELIX_ERR_NO_DEVICE
        if P > 1:
            bwd = abi.DELTA_RULE_BACKWARD_STRUCT.pack(*a, 2, 1.0, *[at] * 15, 1 << 50, *v, *strides)
            assert int(lib.helix_delta_rule_backward_encode(host.handle, None, bwd)) == HELIX_ERR_NO_DEVICE
    host.close()
