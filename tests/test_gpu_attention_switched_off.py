"""Biases of -inf: pairs that they switch off do not count, whatever they leave of a row (the bounds are those of tests/token_bounds.py)."""

import math

import pytest
import torch

from miniworld_b200 import blocks
from tests.token_bounds import attention
from tests.token_reference import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _status():
    yield
    assert blocks.read_status(DEV) == 0


def _run(lengths, h, hk, d, type, table, where, causal, first=1.0, packed=True, mask=None, spare=0, behind=0.0):
    g = torch.Generator(device=DEV).manual_seed(sum(lengths))
    rows = sum(lengths) + spare
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    q, k, v, do = rand(rows, h, d), rand(rows, hk, d), rand(rows, hk, d), 0.1 * rand(rows, h, d)
    v[0] *= first
    for t in (q, k, v, do):
        t[sum(lengths):] = behind
    q, k, v, do = (t.to(type) for t in (q, k, v, do))
    leaves = [q.requires_grad_(True), k.requires_grad_(True), v.requires_grad_(True), table.requires_grad_(True)]
    ends = torch.tensor([0, *lengths]).cumsum(0).to(DEV, torch.int32)
    o = blocks.token_attention(*leaves[:3], offsets=ends, mask=mask, causal=causal, table=table, bucket_of=where)
    got = dict(zip(("o", "q", "k", "v", "table"), (o.detach(), *torch.autograd.grad(o, leaves, do))))
    want, off = attention(*(t.detach() for t in (q, k, v)), do, lengths, mask, causal, None, table.detach(), where)
    for n, t in got.items():
        check(t, want[n], off[n], n)
    return got


@pytest.mark.parametrize("d", [32, 96])
@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
def test_a_token_without_a_key_of_its_own_is_still_a_key(type, d):
    """Causal, the distance 0 switched off in the last head of each group: the first token has no key there, but its value, larger than
    all others, is that of a key for every other row (fp16: the power of two that ds travels times has to cover it)."""
    where = blocks.relative_buckets(4, device=DEV)
    table = 0.3 * torch.randn(9, 4, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    table[4, 1::2] = -math.inf
    got = _run([40, 150], 4, 2, d, type, table, where, True, first=2000.0)
    assert not got["o"][0, 1::2].any() and got["o"][0, 0::2].any()


@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("which", ["first", "last", "all"])
def test_a_head_switched_off_altogether(type, which):
    where = blocks.relative_buckets(2, device=DEV)
    table = torch.zeros(5, 4, device=DEV)
    off = {"first": [0, 2], "last": [1, 3], "all": [0, 1, 2, 3]}[which]
    table[:, off] = -math.inf
    got = _run([129, 60], 4, 2, 64, type, table, where, False, first=500.0)
    assert not got["o"][:, off].any() and not got["q"][:, off].any()


@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
def test_values_that_are_no_key_do_not_count(type):
    """Masked tokens and rows behind the last sequence hold values near the type's greatest: the others' gradients keep their bits."""
    where = blocks.relative_buckets(2, device=DEV)
    rows = 100 + 30 + 20
    mask = torch.arange(rows, device=DEV) % 7 != 3
    table = torch.zeros(5, 2, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    t = [rand(rows, 2, 48).to(type), rand(rows, 1, 48).to(type), rand(rows, 1, 48).to(type), (1e-3 * rand(rows, 2, 48)).to(type)]
    ends = torch.tensor([0, 100, 130], dtype=torch.int32, device=DEV)
    results = []
    for fill in (0.0, 6e4, -6e4):
        for x in t:
            x[~mask] = fill
            x[130:] = fill
        leaves = [x.clone().requires_grad_(True) for x in t[:3]]
        o = blocks.token_attention(*leaves, offsets=ends, mask=mask, table=table, bucket_of=where)
        results.append([o.detach(), *torch.autograd.grad(o, leaves, t[3])])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)
    want, off = attention(*t, [100, 30], mask, False, None, table, where)
    for n, x in zip(("o", "q", "k", "v"), results[-1]):
        check(x, want[n], off[n], n)
