"""The gradients of the attention, the biases' above all, element by element within bounds that a step left out would break
(tests/token_bounds.py, and tests/test_token_bounds.py for what they notice)."""

import pytest
import torch

from miniworld_b200 import blocks
from tests.token_bounds import attention, coherent, flat
from tests.token_reference import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _status():
    yield
    assert blocks.read_status(DEV) == 0


def _gradients(q, k, v, do, lengths, mask, causal, table, where):
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, table)]
    ends = torch.tensor([0, *lengths]).cumsum(0).to(DEV, torch.int32)
    o = blocks.token_attention(*leaves[:3], offsets=ends, mask=mask, causal=causal, table=leaves[3], bucket_of=where)
    return dict(zip(("o", "q", "k", "v", "table"), (o.detach(), *torch.autograd.grad(o, leaves, do))))


def _random(rows, h, hk, d, type, buckets, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    return [t.to(type) for t in (rand(rows, h, d), rand(rows, hk, d), rand(rows, hk, d) + 0.5, 0.1 * rand(rows, h, d))] + [0.5 * rand(buckets, h)]


def _compare(t, lengths, where, mask=None, causal=False, exact=False):
    got = _gradients(*t[:4], lengths, mask, causal, t[4], where)
    want, off = attention(*t[:4], lengths, mask, causal, None, t[4], where, exact)
    for n, x in got.items():
        check(x, want[n], off[n], n)
    return got, want, off


@pytest.mark.parametrize("m,reach", [(640, 32), (700, 8), (700, 255), (1500, 32), (4096, 32)])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
def test_long_sequences(m, reach, type, causal):
    where = blocks.relative_buckets(reach, device=DEV)
    t = _random(m, 2, 1, 32, type, 2 * reach + 1, m)
    _, want, off = _compare(t, [m], where, causal=causal)
    if reach <= 32:  # the bounds bind: what a gradient of zeros is off by is far beyond them
        assert float((want["table"].abs() > off["table"]).double().mean()) > (0.8 if not causal else 0.3)


@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_widths_with_masks_and_packed_sequences(d, causal):
    lengths = [513, 40, 0, 129, 300]
    where = blocks.relative_buckets(128, 8, device=DEV)
    rows = sum(lengths) + 30
    mask = torch.rand(rows, generator=torch.Generator(device=DEV).manual_seed(d), device=DEV) > 0.2
    _compare(_random(rows, 4, 2, d, torch.bfloat16, 32, d), lengths, where, mask, causal)


@pytest.mark.parametrize("m", [512, 1000, 4096])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
def test_the_rounding_of_the_output_stays_out_of_the_biases_gradients(m, type, causal):
    t = flat(m, 32, type, device=DEV)
    _compare(t[:5], [m], t[5], causal=causal, exact=True)


@pytest.mark.parametrize("m", [512, 1000, 4096])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
def test_the_rounding_of_the_probabilities_stays_out_of_the_outer_buckets(m, type, causal):
    t = coherent(m, 32, type, device=DEV)
    _compare(t[:5], [m], t[5], causal=causal)
