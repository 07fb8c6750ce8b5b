"""The table's gradient of the relative position from whole numbers: every sum is exact in fp32, in whatever order, so every pair counts."""

import pytest
import torch

from miniworld_b200 import blocks

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _gradient(dy, rows, index, where, chain=None):
    z = torch.zeros((), device=DEV, dtype=dy.dtype).expand(dy.shape)
    table = torch.zeros(rows, dy.shape[-1], device=DEV, requires_grad=True)
    return torch.autograd.grad(blocks.relative_position(z, table, index, bucket_of=where, chain=chain), table, dy)[0]


@pytest.mark.parametrize("b,n,c", [(2, 1, 64), (3, 31, 16), (2, 33, 130), (2, 203, 64), (1, 300, 101), (1, 257, 1), (4, 64, 256)])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("reach,exact,more", [(32, None, 1), (64, None, 1), (128, None, 1), (255, None, 1), (8, 3, 1), (0, None, 0)])
def test_whole_numbers_are_added_up_exactly(b, n, c, type, reach, exact, more):
    g = torch.Generator(device=DEV).manual_seed(n)
    where = blocks.relative_buckets(reach, exact, device=DEV)
    rows = int(where.max()) + 1 + more
    dy = torch.randint(-3, 4, (b, n, n, c), generator=g, device=DEV).to(type)
    index = torch.randint(0, 2, (b, n), generator=g, device=DEV).cumsum(1)
    chain = torch.arange(n, device=DEV).expand(b, n) // 60 if more else None
    bucket = where.long()[(index[:, None, :] - index[:, :, None]).clamp(-reach, reach) + reach]
    if chain is not None:
        bucket = torch.where(chain[:, None, :] == chain[:, :, None], bucket, rows - 1)
    want = torch.zeros(rows, c, dtype=torch.float64, device=DEV).index_add_(0, bucket.reshape(-1), dy.reshape(-1, c).double())
    assert torch.equal(_gradient(dy, rows, index, where, chain).double(), want)


@pytest.mark.parametrize("n,c,type", [(1500, 64, torch.bfloat16), (4200, 16, torch.bfloat16), (1100, 40, torch.float32)])
def test_ones_are_counted(n, c, type):
    """Counts below 2^24, the pairs of the outer buckets among them."""
    got = _gradient(torch.ones(1, n, n, c, device=DEV, dtype=type), 65, torch.arange(n, device=DEV), blocks.relative_buckets(32, device=DEV))
    far = sum(n - d for d in range(32, n))
    assert far < 1 << 24
    want = torch.tensor([far] + [n - abs(d) for d in range(-31, 32)] + [far], device=DEV).float()
    assert torch.equal(got, want[:, None].expand(-1, c))
