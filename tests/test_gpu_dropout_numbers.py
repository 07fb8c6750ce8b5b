"""The dropout's numbers against the published known answers of Philox-4x32-10, and the module's mask against its key's."""

import pytest
import torch

import miniworld_b200 as mw
from miniworld_b200 import blocks
from tests.test_philox import KNOWN
from tests.token_reference import philox_halves

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _signed(v):
    return v - (1 << 64) if v >> 63 else v


@pytest.mark.parametrize("type", [torch.bfloat16, torch.float32])
def test_known_answers(type):
    """Element 0 .. 7 of a mask stay up to a threshold of their own half, and not at one more."""
    counter, key, words = KNOWN[0]
    halves = [h for w in words for h in (w & 0xFFFF, w >> 16)]
    seed, second = _signed(key[1] << 32 | key[0]), _signed(counter[3] << 32 | counter[2])
    u = torch.ones(8, dtype=type, device=DEV)
    state = torch.tensor([seed, second], device=DEV)
    for i, half in enumerate(halves):
        for threshold, stays in ((half, True), (half + 1, False)):
            y = blocks.block_dropout(None, u, state, p=threshold / 65536)
            assert bool(y[i] != 0) == stays, (i, threshold)


@pytest.mark.parametrize("shared,shape", [(1, (2, 30, 30, 32)), (1, (2, 9, 5, 7)), (None, (3, 40, 24)), (0, (6, 50))])
def test_the_modules_mask_is_its_keys(shared, shape):
    key = torch.tensor([-(2**62) + 12345, 2**61 + 99], device=DEV)
    x, u = torch.randn(shape, device=DEV).bfloat16(), torch.ones(shape, device=DEV, dtype=torch.bfloat16)
    y = mw.BlockDropout(0.25, shared)(x, u, key)
    own = list(shape)
    if shared is not None:
        own[shared] = 1
    count = 1
    for s in own:
        count *= s
    keep = torch.from_numpy(philox_halves(int(key[0]) % 2**64, int(key[1]) % 2**64, count) >= 16384).to(DEV).view(own).expand(shape)
    want = torch.where(keep, (x.double() + 65536 / 49152).to(torch.bfloat16), x)
    assert torch.equal((y != x) & ~keep, torch.zeros_like(keep)) and float((y.double() - want.double()).abs().max()) <= 2.0**-6
    scaled = blocks.block_dropout(None, u, key, p=0.25, shared=shared)
    assert torch.equal(scaled != 0, keep)
