"""Where an infinity or a NaN in each of the delta rule's inputs goes, forward and backward: what it reaches by the formulas, and
what it never does. Everything else keeps its bits."""
import pytest
import torch

from helix_amd.delta import delta_rule, delta_rule_backward

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")
S, HK, H, N, P = 2, 2, 4, 40, 24
HEADS = slice(2, 4)   # of query head 1


def problem(L, dtype):
    gen = torch.Generator().manual_seed(L)
    q, k = (torch.nn.functional.normalize(torch.randn(S, L, HK, N, generator=gen), dim=-1).to(dtype).cuda() for _ in range(2))
    v, do = (torch.randn(S, L, H, P, generator=gen).to(dtype).cuda() for _ in range(2))
    g, beta = (torch.rand(S, L, H, generator=gen).cuda() for _ in range(2))
    s0, ds = (torch.randn(S, H, N, P, generator=gen).cuda() for _ in range(2))
    return {"do": do, "q": q, "k": k, "v": v, "g": -0.2 * g, "beta": beta, "s0": s0, "ds": ds}


def run(p):
    o, s = delta_rule(*(p[n] for n in ("q", "k", "v", "g", "beta", "s0")))
    return dict(zip(("o", "s", "dq", "dk", "dv", "dg", "dbeta", "ds0"), (o, s, *delta_rule_backward(**p))))


def with_one(p, name, at, bad):
    t = p[name].clone()
    t[at] = bad
    return {**p, name: t}


def same_but(got, want, where):
    """Every output has want's bits outside of where[name] (missing: everywhere)."""
    for n in want:
        keep = torch.ones_like(want[n], dtype=torch.bool)
        for at in where.get(n, ()):
            keep[at] = False
        assert torch.equal(got[n][keep], want[n][keep]), n


ALL = slice(None)
KEY_HEAD = {"dq": [(0, ALL, 1)], "dk": [(0, ALL, 1)], "dv": [(0, ALL, HEADS)], "dg": [(0, ALL, HEADS)], "dbeta": [(0, ALL, HEADS)],
            "ds0": [(0, HEADS)]}
VALUE_HEAD = {"dq": [(0, ALL, 1)], "dk": [(0, ALL, 1)], "dv": [(0, ALL, 2)], "dg": [(0, ALL, 2)], "dbeta": [(0, ALL, 2)], "ds0": [(0, 2)]}
COLUMN = {**VALUE_HEAD, "dv": [(0, ALL, 2, 5)], "ds0": [(0, 2, ALL, 5)]}


def first(L, at):
    """The first token whose o may be other: its chunk's, or its own where the call goes token by token."""
    return at if L <= 6 else at // 64 * 64


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("L,at", [(5, 3), (64, 63), (170, 0), (170, 100)])
class TestNotFinite:
    def test_values(self, gpu, L, at, bad, dtype):
        p = problem(L, dtype)
        want, got = run(p), run(with_one(p, "v", (0, at, 2, 5), bad))
        a = first(L, at)
        same_but(got, want, {**VALUE_HEAD, "o": [(0, slice(a, None), 2, 5)], "s": [(0, 2, ALL, 5)], "dv": [], "ds0": []})
        assert not got["o"][0, at:, 2, 5].isfinite().any() and not got["s"][0, 2, :, 5].isfinite().any()
        assert not got["dq"][0, at:, 1].isfinite().any() and not got["dbeta"][0, at, 2].isfinite()

    def test_gradients_of_outputs(self, gpu, L, at, bad, dtype):
        p = problem(L, dtype)
        want, got = run(p), run(with_one(p, "do", (0, at, 2, 5), bad))
        same_but(got, want, COLUMN)
        assert not got["dv"][0, :at + 1, 2, 5].isfinite().any() and not got["ds0"][0, 2, :, 5].isfinite().any()
        assert not got["dq"][0, at, 1].isfinite().any() and not got["dg"][0, :at + 1, 2].isfinite().any()
        assert not got["dbeta"][0, :at + 1, 2].isfinite().any() and not got["dk"][0, :at + 1, 1].isfinite().any()

    def test_queries(self, gpu, L, at, bad, dtype):
        p = problem(L, dtype)
        want, got = run(p), run(with_one(p, "q", (0, at, 1, 3), bad))
        same_but(got, want, {**KEY_HEAD, "o": [(0, at, HEADS)]})
        assert not got["o"][0, at, HEADS].isfinite().any() and not got["dv"][0, :at + 1, HEADS].isfinite().any()
        assert not got["ds0"][0, HEADS].isfinite().all()

    def test_keys(self, gpu, L, at, bad, dtype):
        p = problem(L, dtype)
        want, got = run(p), run(with_one(p, "k", (0, at, 1, 3), bad))
        same_but(got, want, {**KEY_HEAD, "o": [(0, slice(first(L, at), None), HEADS)], "s": [(0, HEADS)]})
        assert not got["o"][0, at:, HEADS].isfinite().any() and not got["s"][0, HEADS].isfinite().all()
        assert not got["dv"][0, :at + 1, HEADS].isfinite().any() and not got["dq"][0, at:, 1].isfinite().any()

    @pytest.mark.parametrize("name", ["g", "beta"])
    def test_gates(self, gpu, name, L, at, bad, dtype):
        if name == "g" and bad == -INF:
            return self.forgets(L, at, dtype)
        p = problem(L, dtype)
        want, got = run(p), run(with_one(p, name, (0, at, 2), bad))
        same_but(got, want, {**VALUE_HEAD, "o": [(0, slice(first(L, at), None), 2)], "s": [(0, 2)]})
        assert not got["o"][0, at:, 2].isfinite().any() and not got["s"][0, 2].isfinite().all()
        assert not got["dq"][0, at:, 1].isfinite().any() and not got["ds0"][0, 2].isfinite().all()

    def forgets(self, L, at, dtype):
        # What was before does not reach what follows, nor the gradients of what follows what was before.
        p = with_one(problem(L, dtype), "g", (0, at, 2), -INF)
        got = run(p)
        assert all(t.isfinite().all() for t in got.values())
        assert (got["ds0"][0, 2] == 0).all() == (at == 0)
        other = dict(p, s0=p["s0"] + 1)
        assert torch.equal(run(other)["s"][0, 2], got["s"][0, 2])

    def test_states(self, gpu, L, at, bad, dtype):
        p = problem(L, dtype)
        want, got = run(p), run(with_one(p, "s0", (0, 2, 3, 5), bad))
        same_but(got, want, {**VALUE_HEAD, "o": [(0, ALL, 2, 5)], "s": [(0, 2, ALL, 5)], "dv": [], "ds0": []})
        assert not got["o"][0, :, 2, 5].isfinite().any() and not got["s"][0, 2, :, 5].isfinite().all()
        want, got = run(p), run(with_one(p, "ds", (0, 2, 3, 5), bad))
        same_but(got, want, COLUMN)
        assert not got["dv"][0, :, 2, 5].isfinite().any() and not got["ds0"][0, 2, :, 5].isfinite().all()
