"""What the delta rule's scratch sizes are for every size that an argument can have, without a GPU."""
import itertools

import pytest

from helix_amd import abi

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
