"""The bounds of tests/token_bounds.py: an imitation of the kernels' roundings keeps them, and one without a step of theirs does not."""

import pytest
import torch

from miniworld_b200 import blocks
from tests.token_bounds import attention, coherent, flat, imitated


def _inputs(m, d, type, seed=0):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    where = blocks.relative_buckets(8)
    return [t.to(type) for t in (rand(m, 2, d), rand(m, 1, d), rand(m, 1, d) + 0.5, 0.1 * rand(m, 2, d))] + [0.5 * rand(17, 2), where]


def _excess(got, want, off):
    return (got - want).abs() - off


@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["random", "flat", "coherent"])
@pytest.mark.parametrize("causal", [False, True])
def test_the_kernels_roundings_keep_the_bounds(type, kind, causal):
    make = {"random": _inputs, "flat": flat, "coherent": coherent}[kind]
    for m in (1, 40, 512):
        q, k, v, do, table, where = make(m, 32, type)
        want, off = attention(q, k, v, do, [m], None, causal, None, table, where, exact=kind == "flat")
        assert float(_excess(imitated(q, k, v, do, m, table, where, causal), want["table"], off["table"]).max()) <= 0


@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
def test_a_delta_from_the_rounded_output_breaks_them(type):
    """Flat probabilities are powers of two, which no rounding changes: what is left is the output's own rounding."""
    q, k, v, do, table, where = flat(512, 32, type)
    want, off = attention(q, k, v, do, [512], None, False, None, table, where, exact=True)
    got = imitated(q, k, v, do, 512, table, where, rest=False)
    inner = slice(1, -1)
    assert float((_excess(got, want["table"], off["table"]) > 0)[inner].double().mean()) > 0.9


@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
def test_outer_buckets_that_keep_the_probabilities_rounding_break_them(type):
    q, k, v, do, table, where = coherent(512, 32, type)
    want, off = attention(q, k, v, do, [512], None, False, None, table, where)
    got = imitated(q, k, v, do, 512, table, where, outer=False)
    excess = _excess(got, want["table"], off["table"])
    assert bool((excess[[0, -1]] > 4 * off["table"][[0, -1]]).all())


@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
def test_a_gradient_of_zeros_breaks_them(type):
    q, k, v, do, table, where = _inputs(512, 32, type)
    want, off = attention(q, k, v, do, [512], None, False, None, table, where)
    assert float((want["table"].abs() > off["table"]).double().mean()) > 0.9
    assert float(off["table"].norm() / want["table"].norm()) < 0.25


def test_the_formulas_are_those_of_differentiation():
    """The float64 gradients against PyTorch's of the same function, with pairs switched off."""
    m, where = 30, blocks.relative_buckets(3)
    g = torch.Generator().manual_seed(5)
    q, k, v, do = (torch.randn(m, n, 8, generator=g, dtype=torch.float64) for n in (4, 2, 2, 4))
    table = torch.randn(7, 4, generator=g, dtype=torch.float64)
    mask = torch.rand(m, generator=g) > 0.2
    leaves = [t.requires_grad_(True) for t in (q, k, v, table)]
    place = torch.arange(m)
    for causal in (False, True):
        bucket = (place[None, :] - place[:, None]).clamp(-3, 3) + 3
        s = torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(2, 1)) * 8**-0.5 + table[bucket].permute(2, 0, 1)
        counts = mask[:, None] & mask[None, :] & ((place[:, None] >= place[None, :]) if causal else True)
        p = torch.where(counts.any(1)[:, None], torch.softmax(s.masked_fill(~counts, -1e300), -1), 0.0) * counts
        o = torch.einsum("hij,jhd->ihd", p, v.repeat_interleave(2, 1))
        grads = torch.autograd.grad(o, leaves, do)
        want, _ = attention(*(t.detach() for t in (q, k, v)), do, [m], mask, causal, None, table.detach(), where)
        for a, b in zip((o.detach(), *grads), (want[n] for n in ("o", "q", "k", "v", "table"))):
            assert float((a - b).abs().max()) < 1e-12
