"""The relative position on the pair tensor against float64 (the sum is rounded once; the table's gradient is a sum in fp32)."""

import pytest
import torch

from miniworld_b200 import blocks
from tests.token_reference import check, half_step, smallest

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _buckets(index, chain, bucket_of, rows):
    reach = bucket_of.numel() // 2
    b = bucket_of.long()[(index[:, None, :] - index[:, :, None]).clamp(-reach, reach) + reach]
    if chain is not None:
        b = torch.where(chain[:, None, :] == chain[:, :, None], b, rows - 1)
    return b


def _compare(b, n, c, type, bucket_of, rows, index, chain=None, fill=None, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    z = torch.randn(b, n, n, c, generator=g, device=DEV).to(type).requires_grad_(True)
    table = torch.randn(rows, c, generator=g, device=DEV).requires_grad_(True)
    dy = torch.randn(b, n, n, c, generator=g, device=DEV).to(type)
    y = blocks.relative_position(z, table, index, bucket_of=bucket_of, chain=chain)
    dz, dt = torch.autograd.grad(y, [z, table], dy)
    bucket = _buckets(index.expand(b, n), None if chain is None else chain.expand(b, n), bucket_of, rows)
    want = z.detach().double() + table.detach().double()[bucket]
    # one rounding of the sum (below 2^-14 the values of fp16 lie 2^-24 apart: half of that), and one of the fp32 sum before it
    check(y, want, (half_step(type) + 2.0**-24) * want.abs() + smallest(type) + 2.0**-24 * (z.detach().abs() + table.detach()[bucket].abs()).double(), "y")
    assert torch.equal(dz, dy)
    sums, size = (torch.zeros(rows, c, dtype=torch.float64, device=DEV).index_add_(0, bucket.reshape(-1), v.reshape(-1, c)) for v in (dy.double(), dy.double().abs()))
    most = torch.bincount(bucket.reshape(-1), minlength=rows).double()[:, None]
    check(dt, sums, 2.0**-24 * size * most.clamp(1, 4096) + 1e-30, "table")
    assert torch.equal(y.detach(), blocks.relative_position(z.detach(), table.detach(), index, bucket_of=bucket_of, chain=chain))
    return dt


def _place(b, n):
    return torch.arange(n, device=DEV).expand(b, n).contiguous()


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 65, 128, 203])
@pytest.mark.parametrize("c", [64, 128])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16, torch.float32])
def test_sizes(n, c, type):
    _compare(2, n, c, type, blocks.relative_buckets(32, device=DEV), 65, _place(2, n))


@pytest.mark.parametrize("c", [1, 2, 3, 8, 20, 63, 65, 101, 130, 256, 384])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float32])
def test_widths(c, type):
    _compare(1, 70, c, type, blocks.relative_buckets(8, device=DEV), 18, _place(1, 70))


@pytest.mark.parametrize("kind", ["random", "same", "backwards", "gaps", "extreme"])
@pytest.mark.parametrize("type", [torch.int32, torch.int64])
def test_any_index_and_chains(kind, type):
    b, n = 3, 90
    g = torch.Generator(device=DEV).manual_seed(1)
    index = {"random": torch.randint(-100, 100, (b, n), generator=g, device=DEV), "same": torch.zeros(b, n, dtype=torch.int64, device=DEV),
             "backwards": _place(b, n).flip(1), "gaps": _place(b, n) * 7 % 61,
             "extreme": torch.where(_place(b, n) % 2 == 0, 2**31 - 1 - _place(b, n), -(2**31) + _place(b, n))}[kind].to(type)
    chain = torch.randint(0, 3, (b, n), generator=g, device=DEV)
    where = blocks.relative_buckets(32, device=DEV)
    if kind == "extreme":  # (the plain form's difference is in 64 bits)
        _compare(b, n, 64, torch.bfloat16, where, 66, index.long(), None)
        _compare(b, n, 64, torch.bfloat16, where, 66, index.long(), chain)
        return
    _compare(b, n, 64, torch.bfloat16, where, 66, index, chain.to(type))
    _compare(b, n, 64, torch.bfloat16, blocks.relative_buckets(128, 8, device=DEV), 33, index, chain)
    _compare(b, n, 128, torch.float32, where, 66, index[:1], chain[:1])  # one for all samples


def test_32_bit_indices_far_apart():
    index = torch.tensor([[2**31 - 1, -(2**31), 0, 5]], dtype=torch.int32, device=DEV)
    z, table = torch.zeros(1, 4, 4, 8, device=DEV), torch.arange(5, device=DEV, dtype=torch.float32)[:, None].repeat(1, 8)
    y = blocks.relative_position(z, table, index, bucket_of=blocks.relative_buckets(2, device=DEV))[0, :, :, 0]
    assert y.tolist() == [[2, 0, 0, 0], [4, 2, 4, 4], [4, 0, 2, 4], [4, 0, 0, 2]]
    far = torch.tensor([[2**63 - 1, -(2**63)]], device=DEV)
    y = blocks.relative_position(z[:, :2, :2].contiguous(), table, far, bucket_of=blocks.relative_buckets(2, device=DEV))[0, :, :, 0]
    assert y.tolist() == [[2, 0], [4, 2]]


@pytest.mark.parametrize("rows", [1, 40, 300, 512])
def test_tables(rows):
    where = torch.randint(0, rows, (101,), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).int()
    _compare(1, 120, 64, torch.bfloat16, where, rows, _place(1, 120), (_place(1, 120) > 50).long())


def test_infinite_gradients_stay_in_their_bucket():
    n, c = 60, 64
    z, table = torch.zeros(1, n, n, c, device=DEV, dtype=torch.bfloat16), torch.zeros(65, c, device=DEV, requires_grad=True)
    dy = torch.ones_like(z)
    dy[0, 3, 7] = float("inf")
    (g,) = torch.autograd.grad(blocks.relative_position(z, table, _place(1, n), bucket_of=blocks.relative_buckets(32, device=DEV)), table, dy)
    assert torch.isinf(g[36]).all() and torch.isfinite(g[:36]).all() and torch.isfinite(g[37:]).all()


def test_leading_dimensions_layouts_and_empty():
    where = blocks.relative_buckets(4, device=DEV)
    z, table = torch.randn(2, 3, 10, 10, 16, device=DEV), torch.randn(9, 16, device=DEV, requires_grad=True)
    y = blocks.relative_position(z, table, torch.arange(10, device=DEV), bucket_of=where)
    assert torch.equal(y[1, 2], blocks.relative_position(z[1, 2], table, torch.arange(10, device=DEV), bucket_of=where))
    assert torch.equal(y.transpose(2, 3).contiguous(), blocks.relative_position(z.transpose(2, 3), table, -torch.arange(10, device=DEV), bucket_of=where))
    odd = torch.empty(z[0, 0].numel() + 1, device=DEV, dtype=torch.bfloat16)[1:].view(10, 10, 16).copy_(z[0, 0])
    assert torch.equal(blocks.relative_position(odd, table, torch.arange(10, device=DEV), bucket_of=where),
                       blocks.relative_position(z[0, 0].bfloat16(), table, torch.arange(10, device=DEV), bucket_of=where))
    for shape in ((0, 5, 5, 16), (2, 0, 0, 16)):
        e = torch.zeros(shape, device=DEV, requires_grad=True)
        y = blocks.relative_position(e, table, torch.zeros(shape[:2], dtype=torch.int64, device=DEV), bucket_of=where)
        assert y.shape == shape and not torch.autograd.grad(y, [e, table], torch.zeros_like(y))[1].any()


def test_bucket_numbers_beyond_the_table_stay_inside():
    where = torch.tensor([-9, 1 << 30, 1], dtype=torch.int32, device=DEV)
    z, table = torch.zeros(1, 20, 20, 8, device=DEV), torch.ones(2, 8, device=DEV, requires_grad=True)
    y = blocks.relative_position(z, table, _place(1, 20), bucket_of=where)
    (g,) = torch.autograd.grad(y.sum(), table)
    assert bool((y == 1).all()) and float(g.sum()) == 20 * 20 * 8


def test_more_than_32_bits_of_elements():
    n, c = 4200, 128  # 2.26e9 elements
    z = torch.zeros(1, n, n, c, device=DEV, dtype=torch.bfloat16)
    table = torch.randn(65, c, device=DEV).bfloat16().float().requires_grad_(True)
    where = blocks.relative_buckets(32, device=DEV)
    y = blocks.relative_position(z, table, _place(1, n), bucket_of=where)
    for i in (0, 1, n // 2, n - 2, n - 1):
        d = (torch.arange(n, device=DEV) - i).clamp(-32, 32) + 32
        assert torch.equal(y.detach()[0, i].float(), table.detach()[d])
    (g,) = torch.autograd.grad(y, table, torch.ones_like(y))
    count = torch.tensor([n - abs(d) for d in range(-31, 32)], device=DEV)
    assert torch.equal(g[1:64, 0], count.float()) and torch.equal(g[:, 0], g[:, c - 1])
    far = sum(n - d for d in range(32, n))
    assert abs(float(g[0, 5]) - far) <= 2.0**-24 * far * 20 and abs(float(g[64, 77]) - far) <= 2.0**-24 * far * 20
