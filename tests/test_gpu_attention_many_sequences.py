"""The biases' gradient over many packed sequences: every tile of every one gives a sum for each distance, and these are added up."""

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


@pytest.mark.parametrize("reach,exact", [(255, None), (256, 128), (32, None)])
def test_many_sequences(reach, exact):
    """A thousand packed sequences of up to five tokens, and a few of several tiles among them."""
    where = blocks.relative_buckets(reach, exact, device=DEV)
    lengths = [(7 * i) % 6 + (300 if i in (10, 999) else 0) for i in range(1000)]
    g = torch.Generator(device=DEV).manual_seed(reach)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    rows = sum(lengths)
    q, k, v, do = (t.bfloat16() for t in (rand(rows, 1, 16), rand(rows, 1, 16), rand(rows, 1, 16) + 0.5, 0.1 * rand(rows, 1, 16)))
    leaves = [q.requires_grad_(True), k.requires_grad_(True), v.requires_grad_(True), (0.5 * rand(int(where.max()) + 1, 1)).requires_grad_(True)]
    o = blocks.token_attention(*leaves[:3], offsets=torch.tensor([0, *lengths]).cumsum(0).to(DEV), table=leaves[3], bucket_of=where)
    got = dict(zip(("o", "q", "k", "v", "table"), (o.detach(), *torch.autograd.grad(o, leaves, do))))
    want, off = attention(*(t.detach() for t in leaves[:3]), do, lengths, table=leaves[3].detach(), bucket_of=where)
    for n, x in got.items():
        check(x, want[n], off[n], n)


@pytest.mark.parametrize("d", [32, 96])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
def test_one_sequence_of_great_gradients_among_many_small_ones(d, type):
    """3000 sequences of two tokens, scores of zero. v = (1, 0) in one channel and dO = (a, 0): ds is a / 4 at distance 0 and -a / 4 at
    distance 1, exactly. a = 2^26 units in the first sequence and 4 in the others: sums of 2^24 and of 2999 ones, which added up one after
    the other in fp32 would stay at 2^24. A sum is made of runs of at most 32 terms in fp32, each addition off by at most 2^-24 of a partial
    sum that is no greater than the whole, 31 of them in the one run that has the great term (the others are exact), of 64-bit sums
    of the runs, and of two more roundings to fp32: 33 2^-24 of the result."""
    n, unit = 3000, 2.0**-12 if type == torch.float16 else 1.0
    where = blocks.relative_buckets(255, device=DEV)
    q = torch.zeros(2 * n, 1, d, dtype=type, device=DEV)
    v, do = q.clone(), q.clone()
    v[0::2, 0, 3] = 1.0
    do[0::2, 0, 3] = 4.0 * unit
    do[0, 0, 3] = 2.0**26 * unit
    table = torch.zeros(511, 1, device=DEV, requires_grad=True)
    ends = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=DEV)
    (got,) = torch.autograd.grad(blocks.token_attention(q, q, v, offsets=ends, table=table, bucket_of=where), table, do)
    want = torch.zeros(511, 1, dtype=torch.float64, device=DEV)
    want[255], want[256] = (2.0**24 + n - 1) * unit, -(2.0**24 + n - 1) * unit
    check(got, want, 33 * 2.0**-24 * want.abs(), "table")
