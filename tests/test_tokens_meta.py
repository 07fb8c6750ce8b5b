"""The token operators' modules on the meta device, and memory that is allocated for them afterwards."""

import copy
import io

import pytest
import torch

import miniworld_b200 as mw
from miniworld_b200 import blocks

MAKE = [lambda: mw.TokenAttention(4), lambda: mw.TokenAttention(4, reach=128, exact=8), lambda: mw.TokenAttention(4, reach=0), lambda: mw.TokenAttention(4, reach=None),
        lambda: mw.RelativePosition(16), lambda: mw.RelativePosition(16, reach=100, exact=20)]


def _same(a, b):
    assert type(a) is type(b) and (a.bucket_of is None) == (b.bucket_of is None)
    if a.bucket_of is not None:
        assert torch.equal(a.bucket_of, b.bucket_of) and a.bucket_of.dtype == torch.int32
    assert {k: (v.shape, v.dtype) for k, v in a.state_dict().items()} == {k: (v.shape, v.dtype) for k, v in b.state_dict().items()}


@pytest.mark.parametrize("make", MAKE)
def test_construction_on_the_meta_device(make):
    with torch.device("meta"):
        m = make()
    assert all(t.is_meta for t in (*m.parameters(), *m.buffers()))
    m = m.to_empty(device="cpu")
    _same(m, make())
    m.load_state_dict(make().state_dict())
    m.reset_parameters()
    if m.table is not None:
        assert m.table.dtype == torch.float32 and bool(torch.isfinite(m.table).all()) and float(m.table.detach().abs().max()) < 1


@pytest.mark.parametrize("make", MAKE)
def test_memory_that_is_allocated_anew(make):
    m = make()
    _same(m.to_empty(device="cpu"), make())
    _same(m.to("meta").to_empty(device="cpu"), make())
    _same(copy.deepcopy(m).to(torch.bfloat16), make())
    file = io.BytesIO()
    torch.save(m, file)
    file.seek(0)
    _same(torch.load(file, weights_only=False), make())
    outer = torch.nn.Sequential(make().to("meta"))
    _same(outer.to_empty(device="cpu")[0], make())


def test_a_map_of_ones_own_stays():
    m = mw.TokenAttention(2, reach=2)
    own = torch.tensor([0, 0, 1, 0, 0], dtype=torch.int32)
    m.bucket_of = own.clone()
    assert torch.equal(m.to(torch.float16).bucket_of, own) and torch.equal(m.to_empty(device="cpu").bucket_of, own)


def test_sizes_of_the_tables():
    for reach, exact, rows in ((32, None, 65), (0, None, 1), (128, 8, 32), (256, 128, 512)):
        assert mw.TokenAttention(2, reach=reach, exact=exact).table.shape == (rows, 2)
        assert int(blocks.relative_buckets(reach, exact).max()) + 1 == rows
    assert mw.RelativePosition(8, reach=32).table.shape == (66, 8)
