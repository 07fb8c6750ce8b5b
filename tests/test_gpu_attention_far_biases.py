"""Finite biases far below all others, as programs write them where a pair is not to count: rows that have no other pairs still attend to
them, and finite biases beyond fp16's range count as its ends."""

import pytest
import torch

from miniworld_b200 import blocks
from tests.token_bounds import attention
from tests.token_reference import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LOW = [-1e4, -65504.0, -1e6, -1e9, -1e30, float(torch.finfo(torch.bfloat16).min), float(torch.finfo(torch.float32).min)]


@pytest.fixture(autouse=True)
def _status():
    yield
    assert blocks.read_status(DEV) == 0


def _run(lengths, d, type, table, where, causal):
    g = torch.Generator(device=DEV).manual_seed(sum(lengths))
    rows, h = sum(lengths), table.shape[1]
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    q, k, v, do = (t.to(type) for t in (rand(rows, h, d), rand(rows, h, d), rand(rows, h, d), rand(rows, h, d)))
    leaves = [t.requires_grad_(True) for t in (q, k, v, table)]
    ends = torch.tensor([0, *lengths]).cumsum(0).to(DEV, torch.int32)
    o = blocks.token_attention(*leaves[:3], offsets=ends, causal=causal, table=table, bucket_of=where)
    got = dict(zip(("o", "q", "k", "v", "table"), (o.detach(), *torch.autograd.grad(o, leaves, do))))
    want, off = attention(*(t.detach() for t in (q, k, v)), do, lengths, None, causal, None, table.detach().clamp(-65504.0, 65504.0), where)
    for n, t in got.items():
        check(t, want[n], off[n], n)
    return got, v.detach(), do


@pytest.mark.parametrize("d", [32, 96])
@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("low", LOW)
@pytest.mark.parametrize("reach", [0, 3, 40])
def test_sequences_of_one_token_whose_own_key_is_low(d, type, low, reach):
    """One key: its probability is one whatever the bias."""
    where = blocks.relative_buckets(reach, device=DEV)
    table = torch.zeros(2 * reach + 1, 2, device=DEV)
    table[reach] = low
    got, v, do = _run([1] * 30, d, type, table, where, False)
    assert torch.equal(got["o"], v) and torch.equal(got["v"], do)


@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("low", LOW)
@pytest.mark.parametrize("causal", [False, True])
def test_no_token_attends_to_itself_where_it_has_others(type, low, causal):
    where = blocks.relative_buckets(3, device=DEV)
    table = 0.5 * torch.randn(7, 2, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    table[3] = low
    got, v, do = _run([1, 2, 3, 40, 200], 64, type, table, where, causal)
    assert torch.equal(got["o"][0], v[0])
    if causal:  # the first token of each has itself only
        firsts = [1, 3, 6, 46]
        assert torch.equal(got["o"][firsts], v[firsts])


@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("low", LOW)
@pytest.mark.parametrize("which", [slice(None), slice(2, 4), slice(0, 3)])
def test_rows_of_low_pairs_only(type, low, which):
    """All distances low in one head, or those that short sequences have."""
    where = blocks.relative_buckets(2, device=DEV)
    table = torch.zeros(5, 2, device=DEV)
    table[which, 1] = low
    _run([2, 2, 3, 150], 48, type, table, where, which == slice(0, 3))


def test_what_is_not_finite_stays():
    q = torch.randn(1, 20, 1, 16, device=DEV).bfloat16()
    where = blocks.relative_buckets(1, device=DEV)
    for bias in (float("nan"), float("inf")):
        table = torch.tensor([[0.0], [bias], [0.0]], device=DEV)
        assert torch.isnan(blocks.token_attention(q, q, q, table=table, bucket_of=where)).all()
